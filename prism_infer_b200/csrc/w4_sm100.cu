// Products with 4-bit weights for many rows, on the 5th-generation tensor cores.
//
// out[r, n] = sum_groups scale[n, g] * sum_{k in g} (code[n, k] - zero[n, g]) * x[r, k]
//
// The weights are the M side: a tile is 128 weight rows by up to 256 activation rows, so one decoding
// of a weight serves 256 rows. Decoded codes are small integers, exact in bf16; the tensor cores sum
// one group's integer products in TMEM (fp32) and the warps that read TMEM apply the group's scale in
// fp32 while the next group's products run. So no weight is rounded, at the price of reading the
// accumulator once per group: (128 x 256) values per group of 128 inputs are 128 packed fp32x2
// multiply-adds per warp scheduler in the 512 cycles that the group's products take.
//
// Warp roles (512 threads, one CTA per SM, persistent over a device-side tile list):
//   warp 0        TMA of the activation rows (64 inputs x 64 rows per copy, 128-byte swizzle)
//   warp 1        TMEM owner and MMA issuer
//   warp 2        bulk copies of packed weights, 128 inputs of 8 row tiles (1 KB each) per slot, and
//                 of their zero points
//   warp 3        bulk copies of scales, 128 inputs of 8 row tiles per slot (their readers run up to
//                 two chunks behind the decoders, so they have a ring of their own)
//   warps 4-7     decode: 16 bytes (four words) per lane and row -> K-major, swizzled bf16 A tile
//   warps 8-15    accumulate: two warps per TMEM lane quarter, each half of the columns; a lane owns
//                 one weight row, so a group's scale is one register
// Stages hold 64 inputs (A 16 KB + B 32 KB, four of them); a stage is full when its copies have
// landed and the four decoding warps have arrived. Two TMEM buffers of 256 columns take turns, one
// group each. Registers are split 40 / 88 / 192 / 192 per thread and warpgroup (512 in all, the launch's 128 x 4).
// Every wait is bounded; one that runs out records PRISM_MOE_ERR_TIMEOUT and the CTA drains its
// copies and MMAs before it frees TMEM.
#include <algorithm>

#include "gemm_sm100.cuh"
#include "internal.h"
#include "w4.cuh"

namespace prism {
namespace {

constexpr int kRowsW = 128;      // weight rows per tile
constexpr int kTok = 256;        // activation rows per tile, at most
constexpr int kTokBox = 64;      // activation rows per copy
constexpr int kAStage = kRowsW * kBK * 2;
constexpr int kBStage = kTok * kBK * 2;
constexpr int kStage = kAStage + kBStage;
constexpr int kNumStages = 4;
constexpr int kPackStage = 8 * 1024;
constexpr int kPackStages = 3;
constexpr int kThreadsW4 = 512;
constexpr int kMaxScaleSlots = 8;
constexpr size_t kPrefixW4 = ((kMaxW4Segments + 1) * 4 + 15) / 16 * 16;

// Shared memory after the stages: packed slots, zero-point slots, scale slots, barriers, prefix.
template <int G>
struct Smem {
  static constexpr int kPG = 128 / G;                 // groups per chunk
  static constexpr int kZeroSlot = kRowsW * kPG;      // bytes
  static constexpr int kScaleSlot = kRowsW * kPG * 2;
  static constexpr int kScaleSlots = kPG == 4 ? 4 : kMaxScaleSlots;
  static constexpr int kPacked = kNumStages * kStage;
  static constexpr int kZeros = kPacked + kPackStages * kPackStage;
  static constexpr int kScales = kZeros + kPackStages * kZeroSlot;
  static constexpr int kBars = kScales + kScaleSlots * kScaleSlot;
  static constexpr int kPrefix = kBars + 320;
  static constexpr int kBytes = 1024 + kPrefix + static_cast<int>(kPrefixW4);
  static_assert(kBytes <= 232448, "shared memory budget");
};

struct LargeParams {
  int num_kb, chunks, tiles, tiles_n;   // 64-input blocks, 128-input chunks, row tiles, M tiles
  int n_out;
  uint16_t* out;
  int64_t rows_cap;
  const int32_t* seg_offsets;
  const int32_t* seg_expert;
  int nseg, num_mats, min_rows;
  const uint8_t *q, *z;
  const uint16_t* s;
  int* err;
  uint64_t wait_ns;
};

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes,
                                          uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void fence_async_smem() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void reg_alloc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void reg_dealloc() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
// (a0, a1) += s * (v0, v1)
__device__ __forceinline__ void fma2(float2& a, uint32_t v0, uint32_t v1, uint64_t s2) {
  uint64_t v, c = *reinterpret_cast<uint64_t*>(&a);
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(v0), "r"(v1));
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(c) : "l"(v), "l"(s2));
  a = *reinterpret_cast<float2*>(&c);
}

// acc[0 .. 32 kBatches) += s * (the accumulator's columns from ``taddr``), 32 columns per wait.
template <int kBatches>
__device__ __forceinline__ void add_scaled(float2 (&acc)[64], uint32_t taddr, float s) {
  const float2 s2 = make_float2(s, s);
  const uint64_t ss = *reinterpret_cast<const uint64_t*>(&s2);
#pragma unroll
  for (int b = 0; b < kBatches; ++b) {
    uint32_t v[2][16];
    tmem_ld16(taddr + b * 32, v[0]);
    tmem_ld16(taddr + b * 32 + 16, v[1]);
    tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 16; ++i)
      fma2(acc[b * 16 + i], v[i >> 3][2 * (i & 7)], v[i >> 3][2 * (i & 7) + 1], ss);
  }
}

struct Tile {
  int sg, e, mt;        // segment, matrix, M tile
  int64_t row0;         // first activation row
  int rows, cols;       // valid activation rows; MMA N (a multiple of 16)
};

__device__ __forceinline__ Tile tile_at(const LargeParams& p, const int32_t* prefix, int64_t item) {
  Tile t;
  const int unit = static_cast<int>(item / p.tiles_n);
  t.mt = static_cast<int>(item % p.tiles_n);
  t.sg = find_segment(prefix, p.nseg, unit);
  const RowSpan span = segment_rows(p.seg_offsets, t.sg, p.rows_cap);
  // a segment's rows in equal parts, each a multiple of 16
  const int parts = prefix[t.sg + 1] - prefix[t.sg];
  const int64_t len = span.end - span.begin;
  const int64_t per = ((len + parts - 1) / parts + 15) / 16 * 16;
  t.row0 = span.begin + (unit - prefix[t.sg]) * per;
  t.rows = static_cast<int>(max(static_cast<int64_t>(0), min(per, span.end - t.row0)));
  t.cols = max(16, (t.rows + 15) / 16 * 16);
  t.e = p.seg_expert ? p.seg_expert[t.sg] : (p.num_mats == 1 ? 0 : t.sg);
  return t;
}

template <int G, bool kZeros, bool kSwiGLU>
__global__ void __launch_bounds__(kThreadsW4, 1)
    w4_large_kernel(const __grid_constant__ CUtensorMap tmap_x, const LargeParams p) {
  using S = Smem<G>;
  constexpr int PG = S::kPG;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* packed = smem + S::kPacked;
  uint8_t* zeros = smem + S::kZeros;
  uint8_t* scales = smem + S::kScales;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kBars);
  uint64_t* empty = full + kNumStages;
  uint64_t* pk_full = empty + kNumStages;
  uint64_t* pk_empty = pk_full + kPackStages;
  uint64_t* sc_full = pk_empty + kPackStages;
  uint64_t* sc_empty = sc_full + kMaxScaleSlots;
  uint64_t* acc_full = sc_empty + kMaxScaleSlots;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* drain = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int32_t* prefix = reinterpret_cast<int32_t*>(smem + S::kPrefix);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kNumStages; ++s) {
      mbar_init(&full[s], 1 + 4);   // the copies' arrival and four decoding warps
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < kPackStages; ++s) {
      mbar_init(&pk_full[s], 1);
      mbar_init(&pk_empty[s], 4);
    }
    for (int i = 0; i < S::kScaleSlots; ++i) {
      mbar_init(&sc_full[i], 1);
      mbar_init(&sc_empty[i], 8);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 8);
    }
    mbar_init(drain, 1);
    *abort = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmap_x);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  if (warp == 2) build_row_blocks(p.seg_offsets, p.nseg, p.rows_cap, kTok, prefix, p.min_rows);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int64_t total = static_cast<int64_t>(prefix[p.nseg]) * p.tiles_n;
  auto give_up = [&]() {
    *abort = 1;
    record_device_error(p.err, PRISM_MOE_ERR_TIMEOUT);
  };
  auto usable = [&](const Tile& t) { return t.e >= 0 && t.e < p.num_mats && t.rows > 0; };

  if (warp < 4) {
    reg_dealloc<40>();
    if (warp == 0 && lane == 0) {
      // ---------------------------------------------------------------- activation rows
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int64_t item = blockIdx.x; ok && item < total; item += gridDim.x) {
        const Tile t = tile_at(p, prefix, item);
        if (!usable(t)) continue;
        const int boxes = (t.cols + kTokBox - 1) / kTokBox;
        for (int kb = 0; kb < p.num_kb; ++kb) {
          if (!mbar_wait_bounded(&empty[stage], phase ^ 1, abort, p.wait_ns)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&full[stage], boxes * kTokBox * kBK * 2);
          uint8_t* b = smem + stage * kStage + kAStage;
          for (int i = 0; i < boxes; ++i)
            tma_load_2d(b + i * kTokBox * kBK * 2, &tmap_x, &full[stage], kb * kBK,
                        static_cast<int32_t>(t.row0) + i * kTokBox);
          if (++stage == kNumStages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      if (!ok) give_up();
    } else if (warp == 1 && lane == 0) {
      // ---------------------------------------------------------------- MMA issuer
      int stage = 0, buf = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int64_t item = blockIdx.x; ok && item < total; item += gridDim.x) {
        const Tile t = tile_at(p, prefix, item);
        if (!usable(t)) continue;
        const uint32_t idesc = idesc_bf16_f32(kRowsW, t.cols);
        for (int kb = 0; ok && kb < p.num_kb; ++kb) {
          if (!mbar_wait_bounded(&full[stage], phase, abort, p.wait_ns)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a0 = smem_u32(smem + stage * kStage), b0 = a0 + kAStage;
#pragma unroll
          for (int kk = 0; kk < kBK / 16; ++kk) {
            // a new group starts: its buffer must have been read
            const bool first = G == 128 ? (kb & 1) == 0 && kk == 0 : (kk * 16) % G == 0;
            if (first) {
              if (!mbar_wait_bounded(&acc_empty[buf], acc_phase ^ 1, abort, p.wait_ns)) {
                ok = false;
                break;
              }
              tc_fence_after();
            }
            tc_mma_bf16(tmem_base + buf * kTok, smem_desc_sw128(a0 + kk * 32),
                        smem_desc_sw128(b0 + kk * 32), idesc, first ? 0u : 1u);
            const bool last = G == 128 ? ((kb & 1) == 1 || kb + 1 == p.num_kb) && kk == 3
                                       : (kk * 16 + 16) % G == 0;
            if (last) {
              tc_commit(&acc_full[buf]);
              buf ^= 1;
              acc_phase ^= buf == 0 ? 1u : 0u;
            }
          }
          if (!ok) break;
          tc_commit(&empty[stage]);
          if (++stage == kNumStages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      if (!ok) give_up();
      if (*abort) {
        tc_commit(drain);   // completes once every MMA issued above has finished
        volatile int never = 0;
        mbar_wait_bounded(drain, 0, &never, kDrainNs);
      }
    } else if (warp == 2) {
      // ---------------------------------------------------------------- packed weights
      int slot = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int64_t item = blockIdx.x; ok && item < total; item += gridDim.x) {
        const Tile t = tile_at(p, prefix, item);
        if (!usable(t)) {
          if (lane == 0 && t.rows > 0) record_device_error(p.err, PRISM_MOE_ERR_ARG);
          continue;
        }
        const int valid = min(8, p.tiles - t.mt * 8);
        const int64_t first = (static_cast<int64_t>(t.e) * p.tiles + t.mt * 8 + lane) * p.chunks;
        for (int c = 0; c < p.chunks; ++c) {
          ok = mbar_wait_bounded(&pk_empty[slot], phase ^ 1, abort, p.wait_ns);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          constexpr int zb = kZeros ? 16 * PG : 0;   // zero points of one row tile
          if (lane == 0) mbar_arrive_expect_tx(&pk_full[slot], valid * (1024 + zb));
          __syncwarp();
          if (lane < valid) {
            bulk_load(packed + slot * kPackStage + lane * 1024, p.q + (first + c) * 1024, 1024,
                      &pk_full[slot]);
            if constexpr (kZeros)
              bulk_load(zeros + slot * S::kZeroSlot + lane * zb, p.z + (first + c) * zb, zb,
                        &pk_full[slot]);
          }
          if (++slot == kPackStages) {
            slot = 0;
            phase ^= 1;
          }
        }
      }
      if (!ok && lane == 0) give_up();
    } else if (warp == 3) {
      // ---------------------------------------------------------------- scales
      int slot = 0;
      uint32_t phase = 0;
      bool ok = true;
      constexpr int bytes = 32 * PG;   // of one row tile and chunk
      for (int64_t item = blockIdx.x; ok && item < total; item += gridDim.x) {
        const Tile t = tile_at(p, prefix, item);
        if (!usable(t)) continue;
        const int valid = min(8, p.tiles - t.mt * 8);
        const int64_t first = (static_cast<int64_t>(t.e) * p.tiles + t.mt * 8 + lane) * p.chunks;
        for (int c = 0; c < p.chunks; ++c) {
          ok = mbar_wait_bounded(&sc_empty[slot], phase ^ 1, abort, p.wait_ns);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          if (lane == 0) mbar_arrive_expect_tx(&sc_full[slot], valid * bytes);
          __syncwarp();
          if (lane < valid)
            bulk_load(scales + slot * S::kScaleSlot + lane * bytes,
                      reinterpret_cast<const uint8_t*>(p.s) + (first + c) * bytes, bytes,
                      &sc_full[slot]);
          if (++slot == S::kScaleSlots) {
            slot = 0;
            phase ^= 1;
          }
        }
      }
      if (!ok && lane == 0) give_up();
    }
  } else if (warp < 8) {
    // ------------------------------------------------------------------ decode
    reg_dealloc<88>();
    const int w = warp - 4, g = lane >> 2, tq = lane & 3;
    const bool odd = g & 1;
    int stage = 0, slot = 0;
    uint32_t phase = 0, pk_phase = 0;
    bool ok = true;
    for (int64_t item = blockIdx.x; ok && item < total; item += gridDim.x) {
      const Tile t = tile_at(p, prefix, item);
      if (!usable(t)) continue;
      for (int c = 0; ok && c < p.chunks; ++c) {
        ok = mbar_wait_bounded(&pk_full[slot], pk_phase, abort, p.wait_ns);
        if (!ok) break;
        // rows g and g + 8 of row tiles 2 w and 2 w + 1
        uint32_t zr[4][PG];
#pragma unroll
        for (int r = 0; r < 4; ++r)
          load_zeros<PG, kZeros>(zeros + slot * S::kZeroSlot,
                                 ((2 * w + (r >> 1)) * 16 + g + 8 * (r & 1)) * PG, zr[r]);
        uint4 v[4];
#pragma unroll
        for (int r = 0; r < 4; ++r)
          v[r] = *reinterpret_cast<const uint4*>(packed + slot * kPackStage + (2 * w + (r >> 1)) * 1024 +
                                                 (r & 1) * 512 + lane * 16);
        __syncwarp();
        if (lane == 0) mbar_arrive(&pk_empty[slot]);
        if (++slot == kPackStages) {
          slot = 0;
          pk_phase ^= 1;
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (2 * c + half >= p.num_kb) break;
          ok = mbar_wait_bounded(&empty[stage], phase ^ 1, abort, p.wait_ns);
          if (!ok) break;
          uint8_t* a = smem + stage * kStage;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int row = (2 * w + (r >> 1)) * 16 + (r & 1) * 8 + g;
            uint8_t* arow = a + (row >> 3) * 1024 + (row & 7) * 128;
            // lanes of odd rows take the two words in the other order: their 16-byte stores then
            // fall into the other half of the banks
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t w0 = word_of(v[r], 2 * half + i), w1 = word_of(v[r], 2 * half + 1 - i);
              const uint32_t word = odd ? w1 : w0;
              const int jj = odd ? 1 - i : i;
              uint32_t zero = zr[r][0];
              if constexpr (PG == 2) zero = zr[r][half];
              if constexpr (PG == 4) zero = odd ? zr[r][2 * half + 1 - i] : zr[r][2 * half + i];
              const uint4 d = make_uint4(code_pair(word, 0, zero), code_pair(word, 1, zero),
                                         code_pair(word, 2, zero), code_pair(word, 3, zero));
              *reinterpret_cast<uint4*>(arow + (((4 * jj + tq) ^ g) << 4)) = d;
            }
          }
          fence_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&full[stage]);
          if (++stage == kNumStages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
    }
    if (!ok) give_up();
  } else {
    // ------------------------------------------------------------------ accumulate
    reg_alloc<192>();
    const int q = warp & 3, side = (warp - 8) >> 2;
    int buf = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    int slot = 0;
    uint32_t sc_phase = 0;
    const int groups = G == 128 ? p.chunks : p.num_kb * (G == 32 ? 2 : 1);
    for (int64_t item = blockIdx.x; ok && item < total; item += gridDim.x) {
      const Tile t = tile_at(p, prefix, item);
      if (!usable(t)) continue;
      const int left = (t.cols / 16 + 1) / 2 * 16;            // columns of side 0
      const int col0 = side ? left : 0, ncols = side ? t.cols - left : left;
      const int row = q * 32 + lane;                          // weight row in the tile
      float2 acc[64];
#pragma unroll
      for (int i = 0; i < 64; ++i) acc[i] = make_float2(0.f, 0.f);
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + col0;
      for (int c = 0; ok && c < p.chunks; ++c) {
        ok = mbar_wait_bounded(&sc_full[slot], sc_phase, abort, p.wait_ns);
        if (!ok) break;
        float sc[PG];
        load_scales<PG>(reinterpret_cast<const uint16_t*>(scales + slot * S::kScaleSlot) + row * PG, sc);
        __syncwarp();
        if (lane == 0) mbar_arrive(&sc_empty[slot]);
        if (++slot == S::kScaleSlots) {
          slot = 0;
          sc_phase ^= 1;
        }
#pragma unroll
        for (int gr = 0; gr < PG; ++gr) {
          if (c * PG + gr >= groups) break;
          ok = mbar_wait_bounded(&acc_full[buf], acc_phase, abort, p.wait_ns);
          if (!ok) break;
          tc_fence_after();
          __syncwarp();
          const uint32_t at = taddr + buf * kTok;
          // few columns, or all 128 of this side (those past ncols hold what an earlier tile left
          // there and are never stored)
          if (ncols > 32)
            add_scaled<4>(acc, at, sc[gr]);
          else if (ncols > 0)
            add_scaled<1>(acc, at, sc[gr]);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&acc_empty[buf]);
          buf ^= 1;
          acc_phase ^= buf == 0 ? 1u : 0u;
        }
      }
      if (!ok) break;
      // ---- output: lanes are consecutive outputs of one activation row
      const int64_t ld = p.n_out;
      if constexpr (kSwiGLU) {
        // lanes 0-7 and 16-23 hold gate rows, the lanes 8 above them the matching up rows; each of a
        // pair finishes one of two columns
        const bool up = lane & 8;
        const int n = (t.mt * kRowsW + q * 32) / 2 + (lane >> 4) * 8 + (lane & 7);
#pragma unroll
        for (int i = 0; i < 64; ++i) {
          if (2 * i >= ncols) break;
          const float got = __shfl_xor_sync(0xffffffffu, up ? acc[i].x : acc[i].y, 8);
          const float h = up ? silu_mul(got, acc[i].y) : silu_mul(acc[i].x, got);
          const int col = col0 + 2 * i + (up ? 1 : 0);
          if (col < t.rows && n < p.n_out) p.out[(t.row0 + col) * ld + n] = float_to_bf16_bits(h);
        }
      } else {
        // neighbours swap a column: each stores two outputs of one row
        const bool second = lane & 1;
        const int n = t.mt * kRowsW + row - (second ? 1 : 0);
#pragma unroll
        for (int i = 0; i < 64; ++i) {
          if (2 * i >= ncols) break;
          const float got = __shfl_xor_sync(0xffffffffu, second ? acc[i].x : acc[i].y, 1);
          const uint32_t d = second ? pack_bf16x2(got, acc[i].y) : pack_bf16x2(acc[i].x, got);
          const int col = col0 + 2 * i + (second ? 1 : 0);
          if (col < t.rows && n < p.n_out)
            *reinterpret_cast<uint32_t*>(p.out + (t.row0 + col) * ld + n) = d;
        }
      }
    }
    if (!ok) give_up();
  }
  tc_fence_before();
  __syncthreads();
  if (*abort) {
    // copies that a given-up wait left in flight land within microseconds: give them a millisecond
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 1000000ull) {
    }
  }
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

template <int G, bool kZeros, bool kSwiGLU>
int launch_large(const CUtensorMap& map, const LargeParams& p, int grid, cudaStream_t st) {
  auto kern = w4_large_kernel<G, kZeros, kSwiGLU>;
  if (int r = ensure_smem_attr(reinterpret_cast<const void*>(kern), Smem<G>::kBytes))
    return r;
  kern<<<grid, kThreadsW4, Smem<G>::kBytes, st>>>(map, p);
  PRISM_LAUNCH_CHECK("w4_large_kernel launch");
  return PRISM_MOE_OK;
}

template <int G>
int launch_group(const CUtensorMap& map, const LargeParams& p, bool swiglu, int grid,
                 cudaStream_t st) {
  if (p.z)
    return swiglu ? launch_large<G, true, true>(map, p, grid, st)
                  : launch_large<G, true, false>(map, p, grid, st);
  return swiglu ? launch_large<G, false, true>(map, p, grid, st)
                : launch_large<G, false, false>(map, p, grid, st);
}

}  // namespace

int w4_product_large(const W4Problem& pr, int min_rows, cudaStream_t st) {
  LargeParams p{};
  p.num_kb = static_cast<int>(ceil_div(pr.K, kBK));
  p.chunks = static_cast<int>(ceil_div(pr.K, 128));
  p.tiles = static_cast<int>(ceil_div(pr.swiglu ? 2 * pr.n_out : pr.n_out, 16));
  p.tiles_n = static_cast<int>(ceil_div(p.tiles, 8));
  p.n_out = static_cast<int>(pr.n_out);
  p.out = static_cast<uint16_t*>(pr.out);
  p.rows_cap = pr.rows_cap;
  p.seg_offsets = pr.seg_offsets;
  p.seg_expert = pr.seg_expert;
  p.nseg = pr.nseg;
  p.num_mats = pr.num_mats;
  p.min_rows = min_rows;
  p.q = static_cast<const uint8_t*>(pr.w.qweight);
  p.s = static_cast<const uint16_t*>(pr.w.scales);
  p.z = static_cast<const uint8_t*>(pr.w.zeros);
  p.err = pr.err;
  p.wait_ns = wait_limit_ns();
  CUtensorMap map;
  const uint64_t dims[2] = {static_cast<uint64_t>(pr.K), static_cast<uint64_t>(pr.rows_cap)};
  const uint64_t strides[1] = {static_cast<uint64_t>(pr.K) * 2};
  const uint32_t box[2] = {kBK, kTokBox};
  if (int r = encode_bf16_map(&map, pr.x, 2, dims, strides, box)) return r;
  const int64_t long_segs = std::min<int64_t>(pr.nseg, pr.rows_cap / (min_rows + 1));
  const int64_t items = (pr.rows_cap / kTok + long_segs) * p.tiles_n;
  const int grid = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(items, num_sms())));
  switch (pr.w.group_size) {
    case 32: return launch_group<32>(map, p, pr.swiglu, grid, st);
    case 64: return launch_group<64>(map, p, pr.swiglu, grid, st);
    default: return launch_group<128>(map, p, pr.swiglu, grid, st);
  }
}

}  // namespace prism
