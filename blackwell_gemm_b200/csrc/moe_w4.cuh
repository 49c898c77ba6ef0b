// Products with 4-bit weights and group scales, one matrix or a bank:
//
//   C[r, n] = sum_k A[r, k] (q[e, n, k] - z[e, n, k / G]) s[e, n, k / G]
//
// with q and z in 0 .. 15 (z = 8 where none are given) and G = 32, 64, 128.
//
// Few rows read every weight for a handful of products each, so they are
// bound by the 4-bit stream from HBM and, close behind, by the integer work of
// unpacking it.  The tensor core takes the rest: warps unpack q - z -- small
// integers, exact in 16 bits -- and these are the MMA's A operand (128 weight
// rows), with the tokens as its N.  A group's product leaves the tensor core as
// fp32 and is multiplied by its scale there, in fp32, on the way into the
// running sum: no weight is ever rounded to 16 bits.  (w4_split_kernel has
// another way to the same end.)
//
// Weights are laid out once (w4_pack_kernel) in records of 128 rows x 128 k,
// in the order a CTA walks them, so a record is one bulk copy and a CTA's
// whole share one sequential read:
//   8192 B  q: [4 t][128 rows][4 c] words, a word being k = 32 c + 8 t .. + 7:
//           its nibbles k = 0, 2, 4, 6 fill the low half and 1, 3, 5, 7 the
//           high half, so one mask gives a pair in order; row r of t stands
//           at place r ^ 2 t (w4_q_offset)
//   scales  [128 / G][128 rows], 16-bit
//   zeros   [128 / G][128 rows], 8-bit, when there are any
//
// Work is divided as in moe_stream.cuh (items are records).  Kernels by the
// rows of a tile: up to 32 with warp-level MMAs (w4_rows_kernel), 64 and 256
// through TMEM (w4_stream_kernel, w4_wide_kernel), 64 and 128 for small groups
// of bf16 (w4_split_kernel).
#pragma once
#include "moe_stream.cuh"

namespace b200 {

constexpr int kW4Rows = 128, kW4K = 128, kW4Q = kW4Rows * kW4K / 2;

__host__ __device__ constexpr int w4_record_bytes(int group, bool zeros) {
  return kW4Q + kW4K / group * kW4Rows * (zeros ? 3 : 2);
}

// Bytes from a record's start to row `row`'s 16 bytes of part t.  The order of
// the rows lets both ways of reading use all banks: 32 rows of one t, or 8
// rows of four.
__host__ __device__ constexpr uint32_t w4_q_offset(int t, int row) {
  return (uint32_t)(t * 2048 + ((row * 16) ^ (t * 32)));
}

// Unpacking.  The logic pipe takes a warp's instruction every other cycle and
// limits this kernel, so a pair of 4-bit values costs one mask and half a
// shift there; the rest is one fused multiply-add on the other pipe.  A
// nibble at bits 0-3 or 4-7 of a 16-bit float is a subnormal (or, with bit 7
// of a bf16, a number of the first binade, which has the same spacing): the
// bits n stand for n 2^-133 (bf16) or n 2^-24 (f16).  Times a power of two
// that is (q - z) kUnit, exactly; finished sums are scaled back by 1 / kUnit.
template <class T>
struct W4Unpack;
template <>
struct W4Unpack<__nv_bfloat16> {
  static constexpr float kUnit = 1.0f / 64;        // 2^-133 x 2^127
  static constexpr uint32_t kLow = 0x7F007F00u;    // 2^127
  static constexpr uint32_t kHigh = 0x7D007D00u;   // 2^123: bits 4-7 count 16
  static __device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t m, uint32_t b) {
    const __nv_bfloat162 r = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&a),
                                     *reinterpret_cast<const __nv_bfloat162*>(&m),
                                     *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ float wide(uint16_t s) {
    return __uint_as_float((uint32_t)s << 16);
  }
};
template <>
struct W4Unpack<__half> {
  static constexpr float kUnit = 1.0f / 512;       // 2^-24 x 2^15
  static constexpr uint32_t kLow = 0x78007800u;    // 2^15
  static constexpr uint32_t kHigh = 0x68006800u;   // 2^11
  static __device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t m, uint32_t b) {
    const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&a),
                              *reinterpret_cast<const __half2*>(&m),
                              *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ float wide(uint16_t s) {
    return __half2float(*reinterpret_cast<const __half*>(&s));
  }
};

// -z kUnit twice, the same way: exact, and no conversion instruction.
template <class T>
__device__ __forceinline__ uint32_t w4_bias(uint32_t z) {
  return W4Unpack<T>::fma2(z * 0x10001u, W4Unpack<T>::kLow ^ 0x80008000u, 0u);
}

// The eight weights of a word, k ascending, two to a register.
template <class T>
__device__ __forceinline__ void w4_pairs(uint32_t w, uint32_t bias, uint32_t* o) {
  using U = W4Unpack<T>;
  const uint32_t v = w >> 8;
  o[0] = U::fma2(w & 0x000F000Fu, U::kLow, bias);
  o[1] = U::fma2(w & 0x00F000F0u, U::kHigh, bias);
  o[2] = U::fma2(v & 0x000F000Fu, U::kLow, bias);
  o[3] = U::fma2(v & 0x00F000F0u, U::kHigh, bias);
}

// D = A B^T (+ D unless `first`) for 16 weight rows, 8 tokens, 16 k, in registers.
template <class T>
__device__ __forceinline__ void mma_16x8x16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                            uint32_t b1, bool first) {
  if constexpr (kFormat<T> == 1) {
    if (first)
      asm volatile(
          "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, "
          "{%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
          : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
          : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
    else
      asm volatile(
          "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, "
          "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
          : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
          : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    if (first)
      asm volatile(
          "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
          "{%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
          : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
          : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
    else
      asm volatile(
          "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
          "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
          : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
          : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}

// A ring stage holds up to two consecutive records of a segment (one bulk
// copy) and the four 64-k slabs of the tile's tokens that go with them (one
// TMA box): the producing thread shares its scheduler with busy warps, and
// with a record and two boxes at a time it fell behind HBM (630 cycles a
// record).
template <int kTok, int kGroup>
struct W4Ring {
  static constexpr int kSub = kW4K / kGroup;               // groups per record
  static constexpr int kSlabRows = kTok;                   // rows of a token box
  static constexpr int kSlab = kSlabRows * 128;
  static constexpr int kTokens = 4 * kSlab;
  static constexpr int kRecords = (2 * w4_record_bytes(kGroup, true) + 1023) / 1024 * 1024;
  static constexpr int kStageBytes = kTokens + kRecords;
  static constexpr int stages(int other) {
    return (214 * 1024 - other) / kStageBytes < 8 ? (214 * 1024 - other) / kStageBytes : 8;
  }
};

// The two copies of a stage.  tmap_t: with K a multiple of 64, the token
// operand as (k in a slab, row, slab), box 64 x kSlabRows x 4; else (k, row),
// box 64 x kSlabRows.
template <class R>
__device__ __forceinline__ void w4_load_tokens(const CUtensorMap* tmap_t, bool slabs, uint32_t dst,
                                               int kb, int row0, uint32_t bar, uint64_t policy) {
  if (slabs) {
    tma_load_3d_hint(dst, tmap_t, 0, row0, 2 * kb, bar, policy);
  } else {
    for (int j = 0; j < 4; ++j)
      tma_load_2d_hint(dst + j * R::kSlab, tmap_t, kb * kW4K + 64 * j, row0, bar, policy);
  }
}
__device__ __forceinline__ const uint8_t* w4_record(const StreamArgs& a, const StreamSegment& s,
                                                    int kb) {
  return a.packed + (long long)s.e * a.expert_bytes +
         ((long long)s.block * a.red_blocks + kb) * a.record_bytes;
}

// Producing thread, both copies into stages of kStageBytes (tokens first), or
// one of them into a ring of its own.
enum W4Part { kW4Both, kW4Weights, kW4Tokens };
template <W4Part kPart, int kTok, int kGroup, int kStages>
__device__ __forceinline__ void w4_produce(const StreamArgs& args, StreamWalk<kTok> walk,
                                           const CUtensorMap* tmap_t, uint32_t ring, uint32_t full,
                                           uint32_t empty, const WaitCtx& wctx) {
  using R = W4Ring<kTok, kGroup>;
  constexpr uint32_t kTokenBytes = kPart == kW4Weights ? 0 : R::kTokens;
  constexpr uint32_t kBytes = kTokenBytes + (kPart == kW4Tokens ? 0 : R::kRecords);
  const uint64_t once = l2_policy_evict_first(), keep = l2_policy_evict_last();
  const bool slabs = args.red % kSlabK == 0;
  uint32_t stage = 0, phase = 0;
  // Looking at a barrier takes 100 cycles and more on a busy SM, so the next
  // stage's is looked at before this stage's copies go out.
  bool ready = true, ok = true;
  long long issued = 0;
  StreamSegment s;
  while (ok && walk.next(&s)) {
    for (int kb = s.kb0; kb < s.kb1; kb += 2) {
      const uint32_t fb = full + stage * 8u;
      const uint32_t sa = ring + stage * kBytes;
      const uint32_t bytes = kPart == kW4Tokens ? 0
                             : kb + 1 < s.kb1   ? 2 * args.record_bytes
                                                : args.record_bytes;
      ok = ready || wait_ready(empty + stage * 8u, phase ^ 1u, wctx, kErrWaitEmpty);
      if (!ok) break;
      if (++stage == kStages) { stage = 0; phase ^= 1u; }
      ready = mbar_test_wait(empty + stage * 8u, phase ^ 1u);
      mbar_arrive_expect_tx(fb, bytes + kTokenBytes);
      if (kPart != kW4Tokens)
        bulk_load_hint(sa + kTokenBytes, w4_record(args, s, kb), bytes, fb, once);
      if (kPart != kW4Weights) w4_load_tokens<R>(tmap_t, slabs, sa, kb, s.row0, fb, keep);
      ++issued;
    }
  }
  drain_copies<kStages>(full, stage, phase, issued, wctx);
}

// Few rows (at most 32 to a tile): unpacked weights go straight from
// registers into warp-level MMAs, without the stores, loads and handshakes of
// the way through TMEM (about half the instructions a record), and with so few
// tokens the tensor core's rate does not matter.  Groups of four warps take
// stages in turn, a warp 32 rows of each record: four groups for up to 8
// tokens, three for 16 (57344 x 8192, 16 tokens: 62.0 us, with four 71.0: a
// thread has 96 registers then, not 128), two for 32.  Some registers are
// spilled in all of them: 24 to 80 bytes stored with 8 tokens, 16 to 108 with
// 16, 68 to 284 with 32.
// 57344 x 8192, groups of 128, takes 48.7 us for one token: 4.9 TB/s of
// packed weights, 0.76 of HBM's measured rate.  Smaller weights take 8 to 14 us
// more than their bytes; no unit is full then (28672 x 8192, 16 tokens: issue
// slots 42 %, tensor pipe 35 %).
// Column n of the products is token (n >> 1) + 4 (n & 1) of its eight, which
// lets eight lanes read all banks of the swizzled token slab.
template <int kTok, int kGroup>
struct W4RowsCfg {
  using Ring = W4Ring<kTok, kGroup>;
  static constexpr int kPitch = 136;  // floats from token to token of the exchange
  static constexpr int kGroups = kTok <= 8 ? 4 : kTok <= 16 ? 3 : 2;
  static constexpr int kExchange = kGroups * kTok * kPitch * 4;
  // Whole turns to a ring, so that a stage is always the same group's: a group
  // tells the laps of a stage apart by one bit, which it can only while it
  // sees every lap (copies may land out of order).
  static constexpr int kStages = Ring::stages(kExchange) / kGroups * kGroups;
  static_assert(kStages >= kGroups, "a stage for each group");
  static constexpr int kThreads = 32 * (4 * kGroups + 1);
  static constexpr int smem_bytes(int experts) {
    return kStages * Ring::kStageBytes + kExchange + group_table_bytes(experts) + 1024;
  }
};

template <int kTok, int kGroup, bool kZeros, class T>
__global__ void __launch_bounds__(W4RowsCfg<kTok, kGroup>::kThreads, 1)
w4_rows_kernel(const __grid_constant__ CUtensorMap tmap_t, const StreamArgs args) {
  using C = W4RowsCfg<kTok, kGroup>;
  using R = typename C::Ring;
  using U = W4Unpack<T>;
  constexpr int kStages = C::kStages;
  constexpr int kSub = R::kSub;
  constexpr int kNt = kTok / 8;
  extern __shared__ uint8_t smem_raw[];
  __shared__ alignas(8) uint64_t bar_full[kStages];
  __shared__ alignas(8) uint64_t bar_empty[kStages];
  __shared__ uint32_t abort_word;

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);  // (warp-uniform)
  const int lane = threadIdx.x & 31;
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t exchange = smem_base + kStages * R::kStageBytes;
  int* s_off = reinterpret_cast<int*>(smem_raw + (exchange + C::kExchange - smem_u32(smem_raw)));
  int* s_tiles = s_off + args.experts + 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(smem_u32(&bar_full[s]), 1);
      mbar_init(smem_u32(&bar_empty[s]), 4);  // one group's warps
    }
    abort_word = 0;
    fence_mbar_init_cluster();
    prefetch_tmap(&tmap_t);
  }
  grid_wait();
  if (warp == 1) stream_groups(args, kTok, s_off, s_tiles);
  __syncthreads();
  grid_launch_next();

  WaitCtx wctx;
  wctx.status = args.status;
  wctx.timeout_ns = args.timeout_ns;
  wctx.abort_local = smem_u32(&abort_word);
  wctx.abort_peer = cluster_map(smem_u32(&abort_word), 0);

  StreamWalk<kTok> walk;
  walk.init(args, s_off, s_tiles);
  StreamSegment s;

  if (warp == 4 * C::kGroups) {
    if (elect_one()) {
      w4_produce<kW4Both, kTok, kGroup, kStages>(args, walk, &tmap_t, smem_base,
                                                 smem_u32(&bar_full[0]), smem_u32(&bar_empty[0]),
                                                 wctx);
    }
    __syncwarp();
    return;
  }
  const int g = lane >> 2, t = lane & 3;
  const int row = (warp & 3) * 32 + g;  // + 0, 8 (first 16 rows), 16, 24 (second)
  const uint32_t group = warp >> 2;
  const int token = (g >> 1) + 4 * (g & 1);  // of column g of each eight
  // bytes of this lane's token row in a slab; 16-byte chunk c at c ^ token
  const uint32_t token_row = token * 128;
  zero_unowned_rows(static_cast<T*>(args.out), args.ldo, args.feat, s_off[0],
                    s_off[args.experts], args.rows,
                    (long long)blockIdx.x * (128 * C::kGroups) + threadIdx.x,
                    gridDim.x * (128ll * C::kGroups));
  uint32_t first_stage = 0, first_phase = 0;  // of the segment
  uint32_t turn = 0;                          // group that takes its first stage
  bool ok = true;
  while (walk.next(&s)) {
    float acc[2][kNt][4];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int n = 0; n < kNt; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[m][n][i] = 0.0f;
    const int stages = (s.kb1 - s.kb0 + 1) / 2;
    const uint32_t offset = group >= turn ? group - turn : group + C::kGroups - turn;
    uint32_t stage = first_stage + offset, phase = first_phase;
    if (stage >= kStages) { stage -= kStages; phase ^= 1u; }
    for (int st = (int)offset; st < stages; st += C::kGroups) {
      const uint32_t bar = smem_u32(&bar_full[stage]);
      if (!__all_sync(0xffffffffu, mbar_test_wait(bar, phase))) {
        int got = 0;
        if (lane == 0) got = wait_ready(bar, phase, wctx, kErrWaitFull);
        ok = __shfl_sync(0xffffffffu, got, 0) != 0;
        __syncwarp();
        if (!ok) break;
      }
      uint32_t tokens = smem_base + stage * R::kStageBytes;
      uint32_t record = tokens + R::kTokens;
      const int records = min(2, s.kb1 - s.kb0 - 2 * st);
#pragma unroll 1
      for (int rec = 0; rec < records;
           ++rec, tokens += 2 * R::kSlab, record += args.record_bytes) {
        uint32_t q[4][4];  // [row][c]
#pragma unroll
        for (int r = 0; r < 4; ++r) ld_shared_v4_u32(record + w4_q_offset(t, row + 8 * r), q[r]);
        float part[2][kNt][4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          constexpr int kPer = kGroup / 32;  // words to a group
          const int sub = c / kPer;
          uint32_t x[kNt][4];
#pragma unroll
          for (int n = 0; n < kNt; ++n)
            ld_shared_v4_u32(tokens + (c >> 1) * R::kSlab + n * 1024 + token_row +
                                 ((((c & 1) * 4 + t) ^ token) << 4),
                             x[n]);
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            uint32_t lo[4], hi[4];
            uint32_t z0 = 8, z1 = 8;
            if constexpr (kZeros) {
              const uint32_t zeros = record + kW4Q + kSub * 256 + sub * 128 + row + 16 * m;
              z0 = ld_shared_u8(zeros);
              z1 = ld_shared_u8(zeros + 8);
            }
            w4_pairs<T>(q[2 * m][c], w4_bias<T>(z0), lo);
            w4_pairs<T>(q[2 * m + 1][c], w4_bias<T>(z1), hi);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t a[4] = {lo[2 * h], hi[2 * h], lo[2 * h + 1], hi[2 * h + 1]};
#pragma unroll
              for (int n = 0; n < kNt; ++n)
                mma_16x8x16<T>(part[m][n], a, x[n][2 * h], x[n][2 * h + 1], c % kPer == 0 && h == 0);
            }
          }
          if (c % kPer == kPer - 1) {
            const uint32_t scales = record + kW4Q + (sub * 128 + row) * 2;
#pragma unroll
            for (int m = 0; m < 2; ++m) {
              const float s0 = U::wide(ld_shared_u16(scales + 32 * m));
              const float s1 = U::wide(ld_shared_u16(scales + 32 * m + 16));
#pragma unroll
              for (int n = 0; n < kNt; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  acc[m][n][i] = fmaf(i < 2 ? s0 : s1, part[m][n][i], acc[m][n][i]);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive_local(smem_u32(&bar_empty[stage]));
      stage += C::kGroups;
      if (stage >= kStages) { stage -= kStages; phase ^= 1u; }
    }
    const uint32_t end = first_stage + stages, laps = end / kStages;
    first_stage = end - laps * kStages;
    first_phase ^= laps & 1u;
    turn = (turn + stages) % C::kGroups;
    // The groups' sums meet in shared memory; warps 0-3 finish the tile,
    // lane = row.
    float* sums = reinterpret_cast<float*>(smem_raw + (exchange - smem_u32(smem_raw)));
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int n = 0; n < kNt; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          sums[(group * kTok + n * 8 + t + 4 * (i & 1)) * C::kPitch + row + 16 * m + 8 * (i >> 1)] =
              acc[m][n][i];
    named_bar_sync(1, 128 * C::kGroups);
    float total[kTok];
    if (warp < 4) {
#pragma unroll
      for (int c = 0; c < kTok; ++c) {
        const float* from = sums + c * C::kPitch + warp * 32 + lane;
        float sum = from[0];
#pragma unroll
        for (int i = 1; i < C::kGroups; ++i) sum += from[i * kTok * C::kPitch];
        total[c] = sum * (1.0f / U::kUnit);
      }
    }
    named_bar_sync(1, 128 * C::kGroups);
    if (warp < 4) {
      const bool valid = __all_sync(0xffffffffu, ok && ld_volatile_shared(wctx.abort_local) == 0);
      stream_finish<kTok, T>(args, walk, s, warp, warp, 0, total, valid);
    }
  }
}

// More rows: through TMEM, 64 tokens to a tile.  Warps: 0 records, 18 tokens
// (each into a ring of its own: a record is free once it is unpacked, its
// tokens when they are multiplied), 1 MMA, 2-9 take the products, 10-17
// unpack.  Two sets unpack the first and the second record of a stage into
// four places of 64 columns.  Products, 64 columns a group and at most two
// groups at a time, go through the other 256 columns, so unpacking, MMAs and
// the scaled sums run beside one another.  Two sets of warps take half of the
// tokens each.  64 rows x 28672 x 8192, groups of 128: 64 us, 1.9 TB/s of
// packed weights; issue slots are 54 % full and the tensor pipe 22 % active:
// a record costs 1200 cycles, the chain of its handshakes.
template <int kGroup>
struct W4Cfg {
  static constexpr int kTok = 64;
  using Ring = W4Ring<kTok, kGroup>;
  static constexpr int kPlaces = 4;                            // records' weights
  static constexpr int kBatch = Ring::kSub < 2 ? 1 : 2;        // groups to a product
  static constexpr int kProducts = 4 / kBatch;
  static constexpr int kTokenStages = 3;
  // Scales wait for their products in a ring of twice as many places: when
  // record j - kPlaces is multiplied, the products of j - 2 kPlaces have been
  // taken (there are never more than kPlaces records between the two).
  static constexpr int kScalePlaces = 2 * kPlaces;
  static constexpr int kScales = kScalePlaces * Ring::kSub * 128 * 2;
  static constexpr int kStages =
      (214 * 1024 - kTokenStages * Ring::kTokens - kScales) / Ring::kRecords;
  static constexpr int kThreads = 32 * (2 + 8 + 8 + 1);
  static constexpr int smem_bytes(int experts) {
    return kTokenStages * Ring::kTokens + kStages * Ring::kRecords + kScales +
           group_table_bytes(experts) + 1024;
  }
};

// tmap_t: as w4_produce takes it.
template <int kGroup, bool kZeros, class T>
__global__ void __launch_bounds__(W4Cfg<kGroup>::kThreads, 1)
w4_stream_kernel(const __grid_constant__ CUtensorMap tmap_t, const StreamArgs args) {
  using C = W4Cfg<kGroup>;
  using R = typename C::Ring;
  using U = W4Unpack<T>;
  constexpr int kTok = C::kTok;
  constexpr int kStages = C::kStages;
  constexpr int kSub = R::kSub;
  extern __shared__ uint8_t smem_raw[];
  __shared__ alignas(8) uint64_t bar_full[kStages];
  __shared__ alignas(8) uint64_t bar_empty[kStages];
  __shared__ alignas(8) uint64_t bar_tok_full[C::kTokenStages];
  __shared__ alignas(8) uint64_t bar_tok_empty[C::kTokenStages];
  __shared__ alignas(8) uint64_t bar_unpacked[C::kPlaces];  // weights are in TMEM
  __shared__ alignas(8) uint64_t bar_used[C::kPlaces];      // their MMAs are done
  __shared__ alignas(8) uint64_t bar_product[C::kProducts]; // a batch of groups is in TMEM
  __shared__ alignas(8) uint64_t bar_taken[C::kProducts];   // it has been read
  __shared__ alignas(8) uint64_t bar_drain;
  __shared__ uint32_t tmem_slot;
  __shared__ uint32_t abort_word;

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);  // (warp-uniform)
  const int lane = threadIdx.x & 31;
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t records = smem_base + C::kTokenStages * R::kTokens;
  const uint32_t scales = records + kStages * R::kRecords;  // [place][group][row], 16-bit
  int* s_off = reinterpret_cast<int*>(smem_raw + (scales + C::kScales - smem_u32(smem_raw)));
  int* s_tiles = s_off + args.experts + 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(smem_u32(&bar_full[s]), 1);
      mbar_init(smem_u32(&bar_empty[s]), 8);  // the unpackers
    }
    for (int s = 0; s < C::kTokenStages; ++s) {
      mbar_init(smem_u32(&bar_tok_full[s]), 1);
      mbar_init(smem_u32(&bar_tok_empty[s]), 1);
    }
    for (int b = 0; b < C::kPlaces; ++b) {
      mbar_init(smem_u32(&bar_unpacked[b]), 4);
      mbar_init(smem_u32(&bar_used[b]), 1);
    }
    for (int b = 0; b < C::kProducts; ++b) {
      mbar_init(smem_u32(&bar_product[b]), 1);
      mbar_init(smem_u32(&bar_taken[b]), 8);
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
  grid_wait();
  if (warp == 2) stream_groups(args, kTok, s_off, s_tiles);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  grid_launch_next();
  const uint32_t tmem_base = tmem_slot;
  const uint32_t tmem_d = tmem_base + C::kPlaces * 64;

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
      w4_produce<kW4Weights, kTok, kGroup, kStages>(args, walk, &tmap_t, records,
                                                    smem_u32(&bar_full[0]),
                                                    smem_u32(&bar_empty[0]), wctx);
    }
    __syncwarp();
  } else if (warp == 18) {
    if (elect_one()) {
      w4_produce<kW4Tokens, kTok, kGroup, C::kTokenStages>(args, walk, &tmap_t, smem_base,
                                                           smem_u32(&bar_tok_full[0]),
                                                           smem_u32(&bar_tok_empty[0]), wctx);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      uint32_t stage = 0, phase = 0;
      uint32_t w = 0, wp = 0, p = 0, pp = 1;  // places in TMEM and their phases
      bool ok = true;
      // (looked at before the MMAs ahead of them go out, as by the producer)
      bool landed = false, unpacked = false, taken = true;
      const uint32_t tok_full = smem_u32(&bar_tok_full[0]), tok_empty = smem_u32(&bar_tok_empty[0]),
                     unpacked0 = smem_u32(&bar_unpacked[0]), used0 = smem_u32(&bar_used[0]),
                     product0 = smem_u32(&bar_product[0]), taken0 = smem_u32(&bar_taken[0]);
      while (ok && walk.next(&s)) {
        const uint32_t idesc = make_idesc_16bit(128, (s.rows + 15) & ~15, kFormat<T>, false, false);
        uint32_t second = 0;
        for (int kb = s.kb0; ok && kb < s.kb1; ++kb) {
          if (!(landed || wait_ready(tok_full + stage * 8u, phase, wctx, kErrWaitFull)) ||
              !(unpacked || wait_ready(unpacked0 + w * 8u, wp, wctx, kErrWaitFull))) {
            ok = false;
            break;
          }
          const uint64_t bdesc =
              make_sdesc_k128(smem_base + stage * R::kTokens + second * 2 * R::kSlab);
          const uint32_t a = tmem_base + w * 64;
          const uint32_t my_tokens = tok_empty + stage * 8u, my_used = used0 + w * 8u;
          const bool last = second != 0 || kb + 1 == s.kb1;  // of its stage
          second = last ? 0u : 1u;
          if (last) {
            if (++stage == C::kTokenStages) { stage = 0; phase ^= 1u; }
          }
          if (++w == C::kPlaces) { w = 0; wp ^= 1u; }
          landed = mbar_test_wait(tok_full + stage * 8u, phase);
          unpacked = mbar_test_wait(unpacked0 + w * 8u, wp);
#pragma unroll
          for (int g = 0; g < kSub / C::kBatch; ++g) {
            if (!taken && !wait_ready(taken0 + p * 8u, pp, wctx, kErrWaitAccEmpty)) {
              ok = false;
              break;
            }
            tc_fence_after_sync();
            const uint32_t d = tmem_d + p * C::kBatch * 64;
            const uint32_t my_product = product0 + p * 8u;
            if (++p == C::kProducts) { p = 0; pp ^= 1u; }
            taken = mbar_test_wait(taken0 + p * 8u, pp);
#pragma unroll
            for (int i = 0; i < C::kBatch * kGroup / kMmaK; ++i) {
              const int k = g * (C::kBatch * kGroup / kMmaK) + i;
              umma_tmem_a_1(d + i * kMmaK / kGroup * 64, a + k * 8,
                            bdesc + ((k >> 2) * R::kSlab + (k & 3) * 32) / 16, idesc,
                            i * kMmaK % kGroup != 0 ? 1u : 0u);
            }
            umma_commit_1(my_product);
          }
          // (with one product to a record its barrier serves the weights too)
          if (C::kProducts != C::kPlaces) umma_commit_1(my_used);
          if (last) umma_commit_1(my_tokens);
        }
      }
      umma_commit_1(smem_u32(&bar_drain));
      if (!mbar_try_wait(smem_u32(&bar_drain), 0))
        wait_slow(smem_u32(&bar_drain), 0, wctx, kErrWaitDrain, false);
    }
    __syncwarp();
  } else {
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    // All lanes look at once (one instruction, one answer); lane 0 waits.
    auto wait_warp = [&](uint32_t bar, uint32_t parity, int code) {
      if (__all_sync(0xffffffffu, mbar_test_wait(bar, parity))) return true;
      int got = 0;
      if (lane == 0) got = wait_ready(bar, parity, wctx, code);
      got = __shfl_sync(0xffffffffu, got, 0);
      __syncwarp();
      return got != 0;
    };
    const uint32_t set = ((uint32_t)(warp - 2) >> 2) & 1u;
    uint32_t stage = 0, phase = 0;
    auto next_stage = [&]() {
      if (++stage == kStages) { stage = 0; phase ^= 1u; }
    };
    bool ok = true;
    if (warp >= 10) {
      // ----------------------------------------------------------- unpack
      uint32_t w = 0, wp = 0, n = 0;
      auto next_place = [&]() {
        if (++w == C::kPlaces) { w = 0; wp ^= 1u; }
        if (++n == C::kScalePlaces) n = 0;
      };
      while (ok && walk.next(&s)) {
        for (int kb = s.kb0; kb < s.kb1; kb += 2, next_stage()) {
          const bool pair = kb + 1 < s.kb1;
          if (set == 1) {
            next_place();
            if (!pair) {
              // Nothing to unpack; the stage still counts this warp.  It waits
              // for the record all the same: a set that did not could come
              // round to the stage again and release it for the other.
              ok = wait_warp(smem_u32(&bar_full[stage]), phase, kErrWaitFull);
              if (!ok) break;
              if (lane == 0) mbar_arrive_local(smem_u32(&bar_empty[stage]));
              continue;
            }
          }
          ok = wait_warp(smem_u32(&bar_full[stage]), phase, kErrWaitFull) &&
               wait_warp(C::kProducts == C::kPlaces ? smem_u32(&bar_product[w % C::kProducts])
                                                    : smem_u32(&bar_used[w]),
                         wp ^ 1u, kErrWaitAccEmpty);
          if (!ok) break;
          tc_fence_after_sync();
          const uint32_t record = records + stage * R::kRecords + set * args.record_bytes;
          uint32_t bias[kSub];
#pragma unroll
          for (int g = 0; g < kSub; ++g)
            bias[g] = w4_bias<T>(
                kZeros ? ld_shared_u8(record + kW4Q + kSub * 256 + g * 128 + row) : 8u);
#pragma unroll
          for (int g = 0; g < kSub; ++g)
            st_shared_u16(scales + ((n * kSub + g) * 128 + row) * 2,
                          ld_shared_u16(record + kW4Q + (g * 128 + row) * 2));
          uint32_t q[4][4];  // [t][c]
#pragma unroll
          for (int t = 0; t < 4; ++t) ld_shared_v4_u32(record + w4_q_offset(t, row), q[t]);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t r[32];
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int t = 0; t < 4; ++t)
                w4_pairs<T>(q[t][2 * h + c], bias[(2 * h + c) * 32 / kGroup], r + c * 16 + t * 4);
            tmem_st_32x32b_x32(tmem_base + w * 64 + h * 32 + lanes, r);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive_local(smem_u32(&bar_empty[stage]));
          tmem_wait_st();
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive_local(smem_u32(&bar_unpacked[w]));
          next_place();
          if (set == 0 && pair) next_place();
        }
      }
    } else {
      // --------------------------------------------------- products, finish
      zero_unowned_rows(static_cast<T*>(args.out), args.ldo, args.feat, s_off[0],
                        s_off[args.experts], args.rows,
                        (long long)blockIdx.x * 256 + (threadIdx.x - 64), gridDim.x * 256ll);
      const int tok0 = (int)set * 32;  // of this warp's tokens
      uint32_t p = 0, pp = 0, n = 0;
      bool ready = false;
      while (walk.next(&s)) {
        float acc[32];
#pragma unroll
        for (int c = 0; c < 32; ++c) acc[c] = 0.0f;
        for (int kb = s.kb0; ok && kb < s.kb1; ++kb) {
          const uint32_t mine = scales + (n * kSub * 128 + row) * 2;
          if (++n == C::kScalePlaces) n = 0;
#pragma unroll 1
          for (int g = 0; g < kSub; g += C::kBatch) {
            ok = ready || wait_warp(smem_u32(&bar_product[p]), pp, kErrWaitAccFull);
            if (!ok) break;
            tc_fence_after_sync();
            float scale[C::kBatch];
#pragma unroll
            for (int j = 0; j < C::kBatch; ++j)
              scale[j] = U::wide(ld_shared_u16(mine + (g + j) * 256));
            const uint32_t d = tmem_d + p * C::kBatch * 64 + tok0 + lanes;
            const uint32_t here = smem_u32(&bar_taken[p]);
            if (++p == C::kProducts) { p = 0; pp ^= 1u; }
            ready = __all_sync(0xffffffffu, mbar_test_wait(smem_u32(&bar_product[p]), pp));
#pragma unroll
            for (int c = 0; c < 32; c += 16) {
              if (tok0 + c < s.rows) {
                uint32_t v[C::kBatch][16];
#pragma unroll
                for (int j = 0; j < C::kBatch; ++j) tmem_ld_32x32b_x16(d + j * 64 + c, v[j]);
                tmem_wait_ld();
#pragma unroll
                for (int j = 0; j < C::kBatch; ++j)
#pragma unroll
                  for (int i = 0; i < 16; ++i)
                    acc[c + i] = fmaf(scale[j], __uint_as_float(v[j][i]), acc[c + i]);
              }
            }
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive_local(here);
          }
        }
#pragma unroll
        for (int c = 0; c < 32; ++c) acc[c] *= 1.0f / U::kUnit;
        const bool valid =
            __all_sync(0xffffffffu, ok && ld_volatile_shared(wctx.abort_local) == 0);
        stream_finish<32, T, 2>(args, walk, s, quarter, (int)set * 4 + quarter, tok0, acc, valid);
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

// More rows, bf16: scaled weights as the sum of two bf16.  w = s (q - z) has 8
// + 4 significant bits.  hi = bf16((q - z) bf16(31/32 s)) is w (1 - 1/32) but
// for two roundings, so lo = w - hi lies between 2^-6 and 2^-3 of w's first
// bit: its bits down to w's last are at most eight, and it is exact.  The sum of
// the two products is the weight's, unrounded; and as lo has w's sign and is
// zero only where w is, a token's infinity comes out as one, not as the NaN of
// inf - inf or inf x 0.  An infinite scale has hi = +-(q - z) and lo = w: their
// sum is w again.  The tensor core works twice, but no group's sums are read
// back: the running sum stays in TMEM to the end of the tile.  (fp16 scales have 11 bits, which two
// fp16 hold as well, but not their range: a weight past 65504, or its low part
// below 2^-24, would be lost.  fp16 takes the kernels above and below.)
// (q - z) carries kUnit here too, which the finished sum gives back; hi + lo is
// w down to scales of 2^-120, below which it loses low bits to bf16's range.
//
// Warps: 0 records, 1 MMA, 2 tokens, 4-11 two sets that take records in turn
// to unpack, 12-15 finish tiles.  kTok 128: two buffers of sums and four half
// records' weights fill TMEM; 64: two and three whole records'.
//
// What bounds it: up to 64 rows a record's unpacking, 1050 cycles (twelve
// packed multiply-adds for eight weights keep their pipe full; a third set of
// warps changed nothing); 128 rows, 1400 to 1600, the tensor pipe 74 % active
// (75 cycles for an MMA of 128 columns with its A in TMEM) and the rest the way
// from unpacked weights to a free place (1700 with two places of whole records).
// 2048 rows x 14336 x 4096, groups of 32: 333 us (0.72 PFLOP/s), where reading
// back each group's sums takes 600.
template <int kTok_, int kGroup>
struct W4SplitCfg {
  static constexpr int kTok = kTok_;
  static constexpr int kSub = kW4K / kGroup;
  static constexpr int kSlab = kTok * 128;
  static constexpr int kTokens = 2 * kSlab;  // a record's
  static constexpr int kTokenStages = 4;
  // A place holds a record's weights or, with fewer columns left, half of
  // them (hi, then lo), so that unpacking and MMAs take turns more finely.
  static constexpr int kParts = kTok == 128 ? 2 : 1;
  static constexpr int kPlace = 128 / kParts;  // columns
  static constexpr int kPlaces = (kTmemCols - 2 * kTok) / kPlace;
  static constexpr int kRecord = (w4_record_bytes(kGroup, true) + 127) / 128 * 128;
  static constexpr int kRoom = (214 * 1024 - kTokenStages * kTokens) / kRecord;
  static constexpr int kStages = kRoom < 12 ? kRoom : 12;
  // Sets of unpacking warps, a record each in turn: no more than places, so
  // that two sets never wait for one place, whose phases they could confuse.
  static constexpr int kSets = 2;
  static_assert(kSets * kParts <= kPlaces && kPlaces % kParts == 0, "one set to a place at a time");
  static constexpr int kThreads = 32 * (8 + 4 * kSets);
  static constexpr int smem_bytes(int experts) {
    return kTokenStages * kTokens + kStages * kRecord + group_table_bytes(experts) + 1024;
  }
};

// hi + lo = p s, two weights at a time; `less`: 31/32 s, or s's sign if that is infinite.
__device__ __forceinline__ void w4_split(uint32_t p, uint32_t s, uint32_t less, uint32_t* hi,
                                         uint32_t* lo) {
  const __nv_bfloat162 a = *reinterpret_cast<const __nv_bfloat162*>(&p);
  const __nv_bfloat162 b = *reinterpret_cast<const __nv_bfloat162*>(&s);
  const __nv_bfloat162 h = __hmul2_rn(a, *reinterpret_cast<const __nv_bfloat162*>(&less));
  const __nv_bfloat162 l = __hfma2(a, b, __hneg2(h));
  *hi = *reinterpret_cast<const uint32_t*>(&h);
  *lo = *reinterpret_cast<const uint32_t*>(&l);
}

// stream_finish for sums that are still in TMEM (`acc`: this warp's lanes,
// first column), 16 columns at a time; `freed` is told when they are read.
template <int kTok>
__device__ __forceinline__ void w4_split_finish(const StreamArgs& a, const StreamWalk<kTok>& walk,
                                                const StreamSegment& s, int quarter, uint32_t acc,
                                                uint32_t freed, bool valid) {
  using T = __nv_bfloat16;
  constexpr float kScale = 1.0f / W4Unpack<T>::kUnit;
  const int lane = threadIdx.x & 31;
  const int f = s.block * 128 + quarter * 32 + lane;
  const bool whole = s.kb0 == 0 && s.kb1 == walk.red_blocks;
  int c0 = blockIdx.x, c1 = blockIdx.x;
  if (!whole) {
    const long long first = s.unit * walk.red_blocks;
    c0 = sk_owner(first, walk.items, walk.ranges);
    c1 = sk_owner(first + walk.red_blocks - 1, walk.items, walk.ranges);
  }
  auto slot = [&](int c) {
    return a.slots + ((long long)c * 2 + (c == c0 ? 1 : 0)) * kTok * 128 + quarter * 32 + lane;
  };
  auto store = [&](int t0, const float (&v)[16]) {
    T* col = static_cast<T*>(a.out) + (long long)(s.row0 + t0) * a.ldo + f;
    const int rows = s.rows - t0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (i < rows && f < a.feat) *col = round_one<T>(v[i] * kScale);
      col += a.ldo;
    }
  };
  tc_fence_after_sync();
  if (valid) {
#pragma unroll 1
    for (int t0 = 0; t0 < s.rows; t0 += 16) {
      uint32_t r[16];
      tmem_ld_32x32b_x16(acc + t0, r);
      tmem_wait_ld();
      float v[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
      if (whole) {
        store(t0, v);
      } else {
        float* to = slot(blockIdx.x) + t0 * 128;
#pragma unroll
        for (int i = 0; i < 16; ++i) __stcg(to + i * 128, v[i]);
      }
    }
  }
  tc_fence_before_sync();
  __syncwarp();
  if (lane == 0) mbar_arrive_local(freed);
  if (whole) return;
  unsigned int before = 0;
  if (lane == 0) before = atomic_add_acq_rel(a.counts + c0 * 16 + quarter, 1u);
  before = __shfl_sync(0xffffffffu, before, 0);
  if (before != (unsigned int)(c1 - c0)) return;
  __syncwarp();
  if (lane == 0) atomicExch(a.counts + c0 * 16 + quarter, 0u);
  if (!valid) return;
#pragma unroll 1
  for (int t0 = 0; t0 < s.rows; t0 += 16) {
    float sum[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) sum[i] = 0.0f;
    // parts in range order, two parts' loads in flight
#pragma unroll 1
    for (int p = c0; p <= c1; p += 2) {
      const float* at = slot(p) + t0 * 128;
      const float* bt = slot(p < c1 ? p + 1 : p) + t0 * 128;
      float v[2][16];
#pragma unroll
      for (int i = 0; i < 16; ++i) v[0][i] = __ldcg(at + i * 128);
#pragma unroll
      for (int i = 0; i < 16; ++i) v[1][i] = p < c1 ? __ldcg(bt + i * 128) : 0.0f;
#pragma unroll
      for (int i = 0; i < 16; ++i) sum[i] += v[0][i];
#pragma unroll
      for (int i = 0; i < 16; ++i) sum[i] += v[1][i];
    }
    store(t0, sum);
  }
}

// tmap_t: the token operand (k, row), box 64 x kTok.
template <int kTok, int kGroup, bool kZeros>
__global__ void __launch_bounds__(W4SplitCfg<kTok, kGroup>::kThreads, 1)
w4_split_kernel(const __grid_constant__ CUtensorMap tmap_t, const StreamArgs args) {
  using T = __nv_bfloat16;
  using C = W4SplitCfg<kTok, kGroup>;
  using U = W4Unpack<T>;
  constexpr int kSub = C::kSub;
  extern __shared__ uint8_t smem_raw[];
  __shared__ alignas(8) uint64_t bar_full[C::kStages];
  __shared__ alignas(8) uint64_t bar_empty[C::kStages];
  __shared__ alignas(8) uint64_t bar_tok_full[C::kTokenStages];
  __shared__ alignas(8) uint64_t bar_tok_empty[C::kTokenStages];
  __shared__ alignas(8) uint64_t bar_unpacked[C::kPlaces];
  __shared__ alignas(8) uint64_t bar_used[C::kPlaces];
  __shared__ alignas(8) uint64_t bar_acc_full[2];
  __shared__ alignas(8) uint64_t bar_acc_empty[2];
  __shared__ alignas(8) uint64_t bar_drain;
  __shared__ uint32_t tmem_slot;
  __shared__ uint32_t abort_word;

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);  // (warp-uniform)
  const int lane = threadIdx.x & 31;
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t records = smem_base + C::kTokenStages * C::kTokens;
  int* s_off = reinterpret_cast<int*>(
      smem_raw + (records + C::kStages * C::kRecord - smem_u32(smem_raw)));
  int* s_tiles = s_off + args.experts + 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(smem_u32(&bar_full[s]), 1);
      mbar_init(smem_u32(&bar_empty[s]), 4);
    }
    for (int s = 0; s < C::kTokenStages; ++s) {
      mbar_init(smem_u32(&bar_tok_full[s]), 1);
      mbar_init(smem_u32(&bar_tok_empty[s]), 1);
    }
    for (int b = 0; b < C::kPlaces; ++b) {
      mbar_init(smem_u32(&bar_unpacked[b]), 4);
      mbar_init(smem_u32(&bar_used[b]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&bar_acc_full[b]), 1);
      mbar_init(smem_u32(&bar_acc_empty[b]), 4);
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
  grid_wait();
  if (warp == 2) stream_groups(args, kTok, s_off, s_tiles);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  grid_launch_next();
  const uint32_t tmem_base = tmem_slot;
  const uint32_t tmem_a = tmem_base + 2 * kTok;

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
      // (weights of a single tile are read once; several tiles come back to them)
      const uint64_t policy =
          s_tiles[args.experts] <= args.experts ? l2_policy_evict_first() : l2_policy_evict_normal();
      uint32_t stage = 0, phase = 0;
      long long issued = 0;
      bool ok = true;
      while (ok && walk.next(&s)) {
        for (int kb = s.kb0; kb < s.kb1; ++kb) {
          ok = wait_ready(smem_u32(&bar_empty[stage]), phase ^ 1u, wctx, kErrWaitEmpty);
          if (!ok) break;
          const uint32_t bar = smem_u32(&bar_full[stage]);
          mbar_arrive_expect_tx(bar, args.record_bytes);
          bulk_load_hint(records + stage * C::kRecord, w4_record(args, s, kb), args.record_bytes,
                         bar, policy);
          ++issued;
          if (++stage == C::kStages) { stage = 0; phase ^= 1u; }
        }
      }
      drain_copies<C::kStages>(smem_u32(&bar_full[0]), stage, phase, issued, wctx);
    }
    __syncwarp();
  } else if (warp == 2) {
    if (elect_one()) {
      const uint64_t policy = l2_policy_evict_last();
      uint32_t stage = 0, phase = 0;
      long long issued = 0;
      bool ok = true;
      while (ok && walk.next(&s)) {
        for (int kb = s.kb0; kb < s.kb1; ++kb) {
          ok = wait_ready(smem_u32(&bar_tok_empty[stage]), phase ^ 1u, wctx, kErrWaitEmpty);
          if (!ok) break;
          const uint32_t bar = smem_u32(&bar_tok_full[stage]);
          mbar_arrive_expect_tx(bar, C::kTokens);
          for (int b = 0; b < 2; ++b)
            tma_load_2d_hint(smem_base + stage * C::kTokens + b * C::kSlab, &tmap_t,
                             kb * kW4K + b * kSlabK, s.row0, bar, policy);
          ++issued;
          if (++stage == C::kTokenStages) { stage = 0; phase ^= 1u; }
        }
      }
      drain_copies<C::kTokenStages>(smem_u32(&bar_tok_full[0]), stage, phase, issued, wctx);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      uint32_t stage = 0, phase = 0, w = 0, wp = 0, buf = 0, bp = 1;
      bool ok = true;
      // (looked at before the MMAs ahead of them go out)
      bool landed = false, unpacked = false;
      const uint32_t tok_full = smem_u32(&bar_tok_full[0]), tok_empty = smem_u32(&bar_tok_empty[0]),
                     unpacked0 = smem_u32(&bar_unpacked[0]), used0 = smem_u32(&bar_used[0]);
      while (ok && walk.next(&s)) {
        const uint32_t idesc = make_idesc_16bit(128, (s.rows + 15) & ~15, kFormat<T>, false, false);
        ok = wait_ready(smem_u32(&bar_acc_empty[buf]), bp, wctx, kErrWaitAccEmpty);
        if (!ok) break;
        const uint32_t d = tmem_base + buf * kTok;
        for (int kb = s.kb0; kb < s.kb1; ++kb) {
          if (!(landed || wait_ready(tok_full + stage * 8u, phase, wctx, kErrWaitFull))) {
            ok = false;
            break;
          }
          const uint64_t bdesc = make_sdesc_k128(smem_base + stage * C::kTokens);
          const uint32_t my_tokens = tok_empty + stage * 8u;
          if (++stage == C::kTokenStages) { stage = 0; phase ^= 1u; }
          landed = mbar_test_wait(tok_full + stage * 8u, phase);
#pragma unroll
          for (int h = 0; h < C::kParts; ++h) {
            if (!(unpacked || wait_ready(unpacked0 + w * 8u, wp, wctx, kErrWaitFull))) {
              ok = false;
              break;
            }
            const uint32_t a = tmem_a + w * C::kPlace;
            const uint32_t my_used = used0 + w * 8u;
            if (++w == C::kPlaces) { w = 0; wp ^= 1u; }
            unpacked = mbar_test_wait(unpacked0 + w * 8u, wp);
            tc_fence_after_sync();
#pragma unroll
            for (int i = 0; i < 8 / C::kParts; ++i) {
              const int k = h * (8 / C::kParts) + i;
              const uint64_t b = bdesc + ((k >> 2) * C::kSlab + (k & 3) * 32) / 16;
              umma_tmem_a_1(d, a + i * 8, b, idesc, k != 0 || kb != s.kb0 ? 1u : 0u);
              umma_tmem_a_1(d, a + C::kPlace / 2 + i * 8, b, idesc, 1u);
            }
            umma_commit_1(my_used);
          }
          if (!ok) break;
          umma_commit_1(my_tokens);
        }
        if (!ok) break;
        umma_commit_1(smem_u32(&bar_acc_full[buf]));
        buf ^= 1u;
        if (buf == 0) bp ^= 1u;
      }
      umma_commit_1(smem_u32(&bar_drain));
      if (!mbar_try_wait(smem_u32(&bar_drain), 0))
        wait_slow(smem_u32(&bar_drain), 0, wctx, kErrWaitDrain, false);
    }
    __syncwarp();
  } else if (warp >= 4) {
    const int quarter = warp & 3;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    auto wait_warp = [&](uint32_t bar, uint32_t parity, int code) {
      if (__all_sync(0xffffffffu, mbar_test_wait(bar, parity))) return true;
      int got = 0;
      if (lane == 0) got = wait_ready(bar, parity, wctx, code);
      got = __shfl_sync(0xffffffffu, got, 0);
      __syncwarp();
      return got != 0;
    };
    bool ok = true;
    if (warp < 4 + 4 * C::kSets) {
      // ----------------------------------------------------------- unpack
      const int row = quarter * 32 + lane;
      const uint32_t set = (uint32_t)(warp - 4) >> 2;
      uint32_t stage = 0, phase = 0, w = 0, wp = 0, turn = 0;
      while (ok && walk.next(&s)) {
        for (int kb = s.kb0; kb < s.kb1; ++kb) {
          if (turn == set) {
            ok = wait_warp(smem_u32(&bar_full[stage]), phase, kErrWaitFull);
            if (!ok) break;
            const uint32_t record = records + stage * C::kRecord;
            uint32_t bias[kSub], scale[kSub], less[kSub];
#pragma unroll
            for (int g = 0; g < kSub; ++g) {
              bias[g] = w4_bias<T>(
                  kZeros ? ld_shared_u8(record + kW4Q + kSub * 256 + g * 128 + row) : 8u);
              scale[g] = ld_shared_u16(record + kW4Q + (g * 128 + row) * 2) * 0x10001u;
              less[g] = (scale[g] & 0x7F80u) == 0x7F80u ? (scale[g] & 0x80008000u) | 0x3F803F80u
                                                        : U::fma2(scale[g], 0x3F783F78u, 0u);
            }
            uint32_t q[4][4];  // [t][c]
#pragma unroll
            for (int t = 0; t < 4; ++t) ld_shared_v4_u32(record + w4_q_offset(t, row), q[t]);
#pragma unroll
            for (int h = 0; h < C::kParts; ++h) {
              ok = ok && wait_warp(smem_u32(&bar_used[w + h]), wp ^ 1u, kErrWaitAccEmpty);
              if (!ok) break;
              tc_fence_after_sync();
              const uint32_t a = tmem_a + (w + h) * C::kPlace + lanes;
#pragma unroll
              for (int j = 0; j < 4 / C::kParts; ++j) {
                const int c = h * (4 / C::kParts) + j;
                uint32_t hi[16], lo[16];
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                  uint32_t v[4];
                  w4_pairs<T>(q[t][c], bias[c * 32 / kGroup], v);
#pragma unroll
                  for (int i = 0; i < 4; ++i)
                    w4_split(v[i], scale[c * 32 / kGroup], less[c * 32 / kGroup], &hi[t * 4 + i],
                             &lo[t * 4 + i]);
                }
                tmem_st_32x32b_x16(a + j * 16, hi);
                tmem_st_32x32b_x16(a + C::kPlace / 2 + j * 16, lo);
              }
              tmem_wait_st();
              tc_fence_before_sync();
              __syncwarp();
              if (lane == 0) {
                mbar_arrive_local(smem_u32(&bar_unpacked[w + h]));
                if (h == C::kParts - 1) mbar_arrive_local(smem_u32(&bar_empty[stage]));
              }
            }
            if (!ok) break;
          }
          if (++turn == C::kSets) turn = 0;
          if (++stage == C::kStages) { stage = 0; phase ^= 1u; }
          w += C::kParts;
          if (w == C::kPlaces) { w = 0; wp ^= 1u; }
        }
      }
    } else {
      // ----------------------------------------------------------- finish
      zero_unowned_rows(static_cast<T*>(args.out), args.ldo, args.feat, s_off[0],
                        s_off[args.experts], args.rows,
                        (long long)blockIdx.x * 128 + (threadIdx.x & 127), gridDim.x * 128ll);
      uint32_t buf = 0, bp = 0;
      while (walk.next(&s)) {
        ok = ok && wait_warp(smem_u32(&bar_acc_full[buf]), bp, kErrWaitAccFull);
        const bool valid =
            __all_sync(0xffffffffu, ok && ld_volatile_shared(wctx.abort_local) == 0);
        w4_split_finish<kTok>(args, walk, s, quarter, tmem_base + buf * kTok + lanes,
                              smem_u32(&bar_acc_empty[buf]), valid);
        buf ^= 1u;
        if (buf == 0) bp ^= 1u;
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

// Many rows: 256 tokens to a tile, so that a record is unpacked once for all
// of them.  A product is one group for one half of the tile's tokens (up to
// 128 columns); three places for products and two for weights fill TMEM.  The
// running sums of 128 weight rows x 256 tokens are half of the SM's registers:
// warps 8-23 hold them, 96 registers to a thread, which warps 0-3 (0 records,
// 1 MMA, 2 tokens) and 4-7 (unpack) leave over; about 100 bytes a thread are
// spilled at the launch's 80.
// What bounds it: a record's tokens, 64 KiB, are written to shared memory and
// read by the MMAs once, which takes it 1100 cycles, and an MMA of 128 columns
// takes about 60 with its A in TMEM; the way from a product's MMAs to its
// place's next use, about 1300 with three places, brings that to 2500
// (2048 rows x 14336 x 4096, groups of 128: 274 us, 0.88 PFLOP/s, in tiles of
// 64 410; groups of 32, four times the products: 605 us, in tiles of 64 802).
template <int kGroup>
struct W4WideCfg {
  static constexpr int kTok = 256;
  static constexpr int kSub = kW4K / kGroup;
  static constexpr int kSlab = kTok * 128;     // 64 k of the tile's tokens
  static constexpr int kBox = 128;             // rows of a token box
  static constexpr int kTokenStages = 5;       // slabs
  static constexpr int kPlaces = 2;            // records' weights
  static constexpr int kProducts = 3;
  // When record j is unpacked the MMAs of j - 2 are done, so all products
  // but the last three before those have been taken: of j - 5 and earlier.
  static constexpr int kScalePlaces = 5;
  static constexpr int kScales = kScalePlaces * kSub * 128 * 2;
  static constexpr int kRecord = (w4_record_bytes(kGroup, true) + 127) / 128 * 128;
  static constexpr int kRoom = (214 * 1024 - kTokenStages * kSlab - kScales) / kRecord;
  static constexpr int kStages = kRoom < 6 ? kRoom : 6;
  static constexpr int kThreads = 768;
  static constexpr int smem_bytes(int experts) {
    return kTokenStages * kSlab + kStages * kRecord + kScales + group_table_bytes(experts) + 1024;
  }
  static_assert(kStages >= 3, "records in flight");
  static_assert((40 + 56) * 128 + 96 * 512 <= kThreads * 80, "registers of the launch");
};

// Tokens of a tile's first half (a multiple of 16 unless it is all of them).
__device__ __forceinline__ int w4_half(int rows) {
  return rows <= 128 ? rows : ((rows + 1) / 2 + 15) & ~15;
}

// stream_finish for the sums that a warp of the wide kernel holds.  Whole
// tiles pass through a slot too: code that holds the sums in registers is
// unrolled, code cold in the instruction cache costs more than the detour
// (a finish of 128 unrolled columns took 29,000 cycles), and what reads them
// back is a short loop.
template <class T>
__device__ __forceinline__ void w4_wide_finish(const StreamArgs& a, const StreamWalk<256>& walk,
                                               const StreamSegment& s, int quarter, int piece,
                                               int h0, const int (&from)[2], const int (&chunks)[2],
                                               const float (&acc)[2][32], bool valid) {
  const int lane = threadIdx.x & 31;
  const int f = s.block * 128 + quarter * 32 + lane;
  const bool whole = s.kb0 == 0 && s.kb1 == walk.red_blocks;
  int c0 = blockIdx.x, c1 = blockIdx.x;
  if (!whole) {
    const long long first = s.unit * walk.red_blocks;
    c0 = sk_owner(first, walk.items, walk.ranges);
    c1 = sk_owner(first + walk.red_blocks - 1, walk.items, walk.ranges);
  }
  // (slots as in stream_finish; a whole tile comes between a CTA's divided
  // ones or instead of one, and slot 2 is its own)
  const int own = whole ? 2 : 0;
  auto slot = [&](int c) {
    return a.slots + ((long long)c * 3 + (own != 0 ? own : c == c0 ? 1 : 0)) * 256 * 128 +
           quarter * 32 + lane;
  };
  if (valid) {
    float* mine = slot(blockIdx.x);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float* to = mine + ((h == 0 ? 0 : h0) + from[h] * 16) * 128;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        if (c < chunks[h]) {
#pragma unroll
          for (int i = 0; i < 16; ++i) __stcg(to + (c * 16 + i) * 128, acc[h][c * 16 + i]);
        }
      }
    }
  }
  __syncwarp();
  if (!whole) {
    unsigned int before = 0;
    if (lane == 0) before = atomic_add_acq_rel(a.counts + c0 * 16 + piece, 1u);
    before = __shfl_sync(0xffffffffu, before, 0);
    if (before != (unsigned int)(c1 - c0)) return;
    __syncwarp();
    if (lane == 0) atomicExch(a.counts + c0 * 16 + piece, 0u);
  }
  if (!valid || f >= a.feat) return;
#pragma unroll 1
  for (int j = 0; j < 4; ++j) {
    const int h = j >> 1;
    if ((j & 1) >= (h == 0 ? chunks[0] : chunks[1])) continue;
    const int t0 = (h == 0 ? from[0] * 16 : h0 + from[1] * 16) + (j & 1) * 16;
    const int rows = s.rows - t0;
    float sum[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) sum[i] = 0.0f;
    // parts in range order
#pragma unroll 1
    for (int p = c0; p <= c1; ++p) {
      const float* at = slot(p) + t0 * 128;
      float v[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = __ldcg(at + i * 128);
#pragma unroll
      for (int i = 0; i < 16; ++i) sum[i] += v[i];
    }
    T* col = static_cast<T*>(a.out) + (long long)(s.row0 + t0) * a.ldo + f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (i < rows) *col = round_one<T>(sum[i] * (1.0f / W4Unpack<T>::kUnit));
      col += a.ldo;
    }
  }
}

// tmap_t: the token operand (k, row), box 64 x 128.
template <int kGroup, bool kZeros, class T>
__global__ void __launch_bounds__(W4WideCfg<kGroup>::kThreads, 1)
w4_wide_kernel(const __grid_constant__ CUtensorMap tmap_t, const StreamArgs args) {
  using C = W4WideCfg<kGroup>;
  using U = W4Unpack<T>;
  constexpr int kTok = C::kTok;
  constexpr int kSub = C::kSub;
  constexpr int kSteps = kGroup / kMmaK;  // MMAs to a product
  extern __shared__ uint8_t smem_raw[];
  __shared__ alignas(8) uint64_t bar_full[C::kStages];
  __shared__ alignas(8) uint64_t bar_empty[C::kStages];
  __shared__ alignas(8) uint64_t bar_tok_full[C::kTokenStages];
  __shared__ alignas(8) uint64_t bar_tok_empty[C::kTokenStages];
  __shared__ alignas(8) uint64_t bar_unpacked[C::kPlaces];
  __shared__ alignas(8) uint64_t bar_used[C::kPlaces];
  __shared__ alignas(8) uint64_t bar_product[C::kProducts];
  __shared__ alignas(8) uint64_t bar_taken[C::kProducts];
  __shared__ alignas(8) uint64_t bar_drain;
  __shared__ uint32_t tmem_slot;
  __shared__ uint32_t abort_word;

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);  // (warp-uniform)
  const int lane = threadIdx.x & 31;
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t records = smem_base + C::kTokenStages * C::kSlab;
  const uint32_t scales = records + C::kStages * C::kRecord;  // [place][group][row], 16-bit
  int* s_off = reinterpret_cast<int*>(smem_raw + (scales + C::kScales - smem_u32(smem_raw)));
  int* s_tiles = s_off + args.experts + 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(smem_u32(&bar_full[s]), 1);
      mbar_init(smem_u32(&bar_empty[s]), 4);
    }
    for (int s = 0; s < C::kTokenStages; ++s) {
      mbar_init(smem_u32(&bar_tok_full[s]), 1);
      mbar_init(smem_u32(&bar_tok_empty[s]), 1);
    }
    for (int b = 0; b < C::kPlaces; ++b) {
      mbar_init(smem_u32(&bar_unpacked[b]), 4);
      mbar_init(smem_u32(&bar_used[b]), 1);
    }
    for (int b = 0; b < C::kProducts; ++b) {
      mbar_init(smem_u32(&bar_product[b]), 1);
      mbar_init(smem_u32(&bar_taken[b]), 16);
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
  grid_wait();
  if (warp == 2) stream_groups(args, kTok, s_off, s_tiles);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  grid_launch_next();
  const uint32_t tmem_base = tmem_slot;
  const uint32_t tmem_a = tmem_base + C::kProducts * 128;

  WaitCtx wctx;
  wctx.status = args.status;
  wctx.timeout_ns = args.timeout_ns;
  wctx.abort_local = smem_u32(&abort_word);
  wctx.abort_peer = wctx.abort_local;

  StreamWalk<kTok> walk;
  walk.init(args, s_off, s_tiles);
  StreamSegment s;

  if (warp < 4) {
    registers_dec<40>();
    if (warp == 0) {
      if (elect_one()) {
        const uint64_t policy = l2_policy_evict_normal();
        uint32_t stage = 0, phase = 0;
        long long issued = 0;
        bool ok = true;
        while (ok && walk.next(&s)) {
          for (int kb = s.kb0; kb < s.kb1; ++kb) {
            ok = wait_inline(smem_u32(&bar_empty[stage]), phase ^ 1u, wctx, kErrWaitEmpty);
            if (!ok) break;
            const uint32_t bar = smem_u32(&bar_full[stage]);
            mbar_arrive_expect_tx(bar, args.record_bytes);
            bulk_load_hint(records + stage * C::kRecord, w4_record(args, s, kb), args.record_bytes,
                           bar, policy);
            ++issued;
            if (++stage == C::kStages) { stage = 0; phase ^= 1u; }
          }
        }
        drain_copies<C::kStages>(smem_u32(&bar_full[0]), stage, phase, issued, wctx);
      }
    } else if (warp == 2) {
      if (elect_one()) {
        const uint64_t policy = l2_policy_evict_last();
        uint32_t stage = 0, phase = 0;
        long long issued = 0;
        bool ok = true;
        while (ok && walk.next(&s)) {
          const int boxes = s.rows > C::kBox ? 2 : 1;
          for (int kb = 2 * s.kb0; kb < 2 * s.kb1; ++kb) {
            ok = wait_inline(smem_u32(&bar_tok_empty[stage]), phase ^ 1u, wctx, kErrWaitEmpty);
            if (!ok) break;
            const uint32_t bar = smem_u32(&bar_tok_full[stage]);
            mbar_arrive_expect_tx(bar, boxes * C::kBox * 128);
            for (int b = 0; b < boxes; ++b)
              tma_load_2d_hint(smem_base + stage * C::kSlab + b * C::kBox * 128, &tmap_t,
                               kb * kSlabK, s.row0 + b * C::kBox, bar, policy);
            ++issued;
            if (++stage == C::kTokenStages) { stage = 0; phase ^= 1u; }
          }
        }
        drain_copies<C::kTokenStages>(smem_u32(&bar_tok_full[0]), stage, phase, issued, wctx);
      }
    } else if (warp == 1) {
      if (elect_one()) {
        uint32_t stage = 0, phase = 0;               // token slabs
        uint32_t w = 0, wp = 0, p = 0, pp = 1;       // places in TMEM and their phases
        bool ok = true;
        // (looked at before the MMAs ahead of them go out)
        bool landed = false, unpacked = false, taken = true;
        const uint32_t tok_full = smem_u32(&bar_tok_full[0]), unpacked0 = smem_u32(&bar_unpacked[0]),
                       taken0 = smem_u32(&bar_taken[0]);
        const uint32_t to_empty = smem_u32(&bar_tok_empty[0]) - tok_full,
                       to_used = smem_u32(&bar_used[0]) - unpacked0,
                       to_product = smem_u32(&bar_product[0]) - taken0;
        while (ok && walk.next(&s)) {
          const int h0 = w4_half(s.rows);
          const bool two = s.rows > h0;
          const uint32_t idesc0 = make_idesc_16bit(128, (h0 + 15) & ~15, kFormat<T>, false, false);
          const uint32_t idesc1 =
              make_idesc_16bit(128, (s.rows - h0 + 15) & ~15, kFormat<T>, false, false);
          for (int left = s.kb1 - s.kb0; left > 0; --left) {
            const uint32_t a = tmem_a + w * 64;
            const uint32_t my_unpacked = unpacked0 + w * 8u;
            if (!unpacked && !wait_inline(my_unpacked, wp, wctx, kErrWaitFull)) {
              ok = false;
              break;
            }
            if (++w == C::kPlaces) { w = 0; wp ^= 1u; }
            unpacked = mbar_test_wait(unpacked0 + w * 8u, wp);
            uint32_t slab[2];
#pragma unroll
            for (int g = 0; g < kSub; ++g) {
              // the slabs that this group begins
#pragma unroll
              for (int j = 0; j < 2; ++j)
                if (j * 4 >= g * kSteps && j * 4 < (g + 1) * kSteps) {
                  slab[j] = stage;
                  if (!landed && !wait_inline(tok_full + stage * 8u, phase, wctx, kErrWaitFull))
                    ok = false;
                  if (++stage == C::kTokenStages) { stage = 0; phase ^= 1u; }
                  landed = mbar_test_wait(tok_full + stage * 8u, phase);
                }
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                if (h == 1 && !two) break;
                const uint32_t my_taken = taken0 + p * 8u;
                if (!taken && !wait_inline(my_taken, pp, wctx, kErrWaitAccEmpty)) ok = false;
                if (!ok) break;
                const uint32_t d = tmem_base + p * 128;
                if (++p == C::kProducts) { p = 0; pp ^= 1u; }
                taken = mbar_test_wait(taken0 + p * 8u, pp);
                tc_fence_after_sync();
                const uint32_t first = smem_base + (h == 0 ? 0u : (uint32_t)h0 * 128u);
#pragma unroll
                for (int i = 0; i < kSteps; ++i) {
                  const int k = g * kSteps + i;
                  umma_tmem_a_1(d, a + k * 8,
                                make_sdesc_k128(first + slab[k >> 2] * C::kSlab) + (k & 3) * 2,
                                h == 0 ? idesc0 : idesc1, i != 0 ? 1u : 0u);
                }
                umma_commit_1(my_taken + to_product);
              }
              if (!ok) break;
#pragma unroll
              for (int j = 0; j < 2; ++j)
                if (j * 4 + 4 > g * kSteps && j * 4 + 4 <= (g + 1) * kSteps)
                  umma_commit_1(tok_full + to_empty + slab[j] * 8u);
            }
            if (!ok) break;
            umma_commit_1(my_unpacked + to_used);
          }
        }
        umma_commit_1(smem_u32(&bar_drain));
        wait_inline(smem_u32(&bar_drain), 0, wctx, kErrWaitDrain, true);
      }
    }
    __syncwarp();
    tc_fence_before_sync();
    named_bar_sync(1, C::kThreads);
    if (warp == 1) {
      tc_fence_after_sync();
      tmem_dealloc_1(tmem_base, kTmemCols);
    }
  } else {
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    auto wait_warp = [&](uint32_t bar, uint32_t parity, int code) {
      if (__all_sync(0xffffffffu, mbar_test_wait(bar, parity))) return true;
      int got = 0;
      if (lane == 0) got = wait_inline(bar, parity, wctx, code);
      got = __shfl_sync(0xffffffffu, got, 0);
      __syncwarp();
      return got != 0;
    };
    bool ok = true;
    if (warp < 8) {
      // ----------------------------------------------------------- unpack
      registers_dec<56>();
      uint32_t stage = 0, phase = 0, w = 0, wp = 0, n = 0;
      while (ok && walk.next(&s)) {
        for (int kb = s.kb0; kb < s.kb1; ++kb) {
          ok = wait_warp(smem_u32(&bar_full[stage]), phase, kErrWaitFull);
          if (!ok) break;
          const uint32_t record = records + stage * C::kRecord;
          uint32_t bias[kSub], scale[kSub];
#pragma unroll
          for (int g = 0; g < kSub; ++g) {
            bias[g] = w4_bias<T>(
                kZeros ? ld_shared_u8(record + kW4Q + kSub * 256 + g * 128 + row) : 8u);
            scale[g] = ld_shared_u16(record + kW4Q + (g * 128 + row) * 2);
          }
          uint32_t q[4][4];  // [t][c]
#pragma unroll
          for (int t = 0; t < 4; ++t) ld_shared_v4_u32(record + w4_q_offset(t, row), q[t]);
          ok = wait_warp(smem_u32(&bar_used[w]), wp ^ 1u, kErrWaitAccEmpty);
          if (!ok) break;
          tc_fence_after_sync();
#pragma unroll
          for (int g = 0; g < kSub; ++g)
            st_shared_u16(scales + ((n * kSub + g) * 128 + row) * 2, (uint16_t)scale[g]);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t r[16];
#pragma unroll
            for (int t = 0; t < 4; ++t) w4_pairs<T>(q[t][c], bias[c * 32 / kGroup], r + t * 4);
            tmem_st_32x32b_x16(tmem_a + w * 64 + c * 16 + lanes, r);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive_local(smem_u32(&bar_empty[stage]));
          tmem_wait_st();
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive_local(smem_u32(&bar_unpacked[w]));
          if (++stage == C::kStages) { stage = 0; phase ^= 1u; }
          if (++w == C::kPlaces) { w = 0; wp ^= 1u; }
          if (++n == C::kScalePlaces) n = 0;
        }
      }
    } else {
      // --------------------------------------------------- products, finish
      registers_inc<96>();
      const int set = (warp - 8) >> 2;  // takes a fourth of each product's columns
      zero_unowned_rows(static_cast<T*>(args.out), args.ldo, args.feat, s_off[0],
                        s_off[args.experts], args.rows,
                        (long long)blockIdx.x * 512 + (threadIdx.x - 256), gridDim.x * 512ll);
      uint32_t p = 0, pp = 0, n = 0;
      while (walk.next(&s)) {
        const int h0 = w4_half(s.rows);
        // this warp's columns of a half: up to two chunks of 16 from from[h] on
        int from[2], chunks[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int all = ((h == 0 ? h0 : s.rows - h0) + 15) >> 4;
          from[h] = all * set >> 2;
          chunks[h] = (all * (set + 1) >> 2) - from[h];
        }
        float acc[2][32];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int c = 0; c < 32; ++c) acc[h][c] = 0.0f;
        for (int kb = s.kb0; ok && kb < s.kb1; ++kb) {
          const uint32_t mine = scales + (n * kSub * 128 + row) * 2;
          if (++n == C::kScalePlaces) n = 0;
#pragma unroll 1
          for (int g = 0; g < kSub; ++g) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (h == 1 && s.rows <= h0) break;
              ok = ok && wait_warp(smem_u32(&bar_product[p]), pp, kErrWaitAccFull);
              if (!ok) break;
              tc_fence_after_sync();
              const float scale = U::wide(ld_shared_u16(mine + g * 256));
              const uint32_t d = tmem_base + p * 128 + from[h] * 16 + lanes;
              // (a second chunk that is another warp's is read and not used)
              if (chunks[h] > 0) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                  uint32_t v[16];
                  tmem_ld_32x32b_x16(d + c * 16, v);
                  tmem_wait_ld();
#pragma unroll
                  for (int i = 0; i < 16; ++i)
                    acc[h][c * 16 + i] =
                        fmaf(scale, __uint_as_float(v[i]), acc[h][c * 16 + i]);
                }
              }
              tc_fence_before_sync();
              __syncwarp();
              if (lane == 0) mbar_arrive_local(smem_u32(&bar_taken[p]));
              if (++p == C::kProducts) { p = 0; pp ^= 1u; }
            }
          }
        }
        const bool valid =
            __all_sync(0xffffffffu, ok && ld_volatile_shared(wctx.abort_local) == 0);
        w4_wide_finish<T>(args, walk, s, quarter, set * 4 + quarter, h0, from, chunks, acc, valid);
      }
    }
    tc_fence_before_sync();
    named_bar_sync(1, C::kThreads);
  }
}

// q: experts x N x K / 2 bytes, the low nibble the even k; scales, zeros:
// experts x N x K / group, 16-bit and 8-bit; all contiguous.  One block per
// record; rows and k past the matrix get scale 0 and q = 8.  A zero point above
// 15 is reported in the device's error word.
__global__ void __launch_bounds__(256)
w4_pack_kernel(const uint8_t* q, const uint16_t* scales, const uint8_t* zeros, uint8_t* out, int N,
               int K, int group, int blocks, int red_blocks, int record_bytes, int* status) {
  grid_wait();
  grid_launch_next();
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
    *reinterpret_cast<uint32_t*>(dst + w4_q_offset(word & 3, row) + (word >> 2) * 4) = w;
  }
  const int sub = kW4K / group, groups = K / group;
  for (int i = threadIdx.x; i < kW4Rows * sub; i += blockDim.x) {
    const int row = i / sub, g = i - row * sub;
    const int n = block * kW4Rows + row, kg = kb * sub + g;
    const bool in = n < N && kg < groups;
    const long long at = (e * N + n) * (long long)groups + kg;
    reinterpret_cast<uint16_t*>(dst + kW4Q)[g * 128 + row] = in ? scales[at] : (uint16_t)0;
    if (zeros != nullptr) {
      const uint32_t z = in ? zeros[at] : 8u;
      if (z > 15u) atomicCAS(status, 0, kErrZeroPoint);
      dst[kW4Q + sub * 256 + g * 128 + row] = z & 15u;
    }
  }
}

}  // namespace b200
