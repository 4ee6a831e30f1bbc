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
// Warp roles (persistent over a device-side tile list):
//   warp 0        TMA of the activation rows (64 inputs x 64 rows per copy, 128-byte swizzle)
//   warp 1        TMEM owner and MMA issuer
//   warp 2        TMA of packed weights, 128 inputs of 8 row tiles (1 KB each) per copy, and of their
//                 zero points
//   warp 3        TMA of scales, 128 inputs of 8 row tiles per copy (their readers run up to two
//                 chunks behind the decoders, so they have a ring of their own)
//                 These four run their loops as whole warps and elect a lane for the copy or MMA, so
//                 that its operands are uniform registers; in a one-lane branch each had to be moved
//                 there, and issuing a stage took longer than its products.
//   warps 4-7     decode: 16 bytes (four words) per lane and row -> K-major, swizzled bf16 A tile
//   warps 8-15    accumulate (8-11 for tiles of 64 rows): two warps per TMEM lane quarter, each half of the
//                 columns; a lane owns one weight row, so a group's scale is one register
// Stages hold 64 inputs (wide tiles: A 16 KB + B 32 KB, four of them); a stage is full when its copies
// have landed and the four decoding warps have arrived. TMEM buffers (two of 256 columns) take turns,
// one group each. Registers are split per warpgroup (Shape).
//
// What bounds it: with groups of 128 a chunk of 128 inputs takes a wide tile about 1450 cycles where
// its eight MMAs need 1024; the accumulating warps' TMEM loads and multiply-adds are nearly as long,
// and four reads of the accumulator per chunk bound groups of 32. A tile's output adds about 5400 cycles
// in which the MMAs stand (no third TMEM buffer fits).
// Measured: 8192 x 4736 x 4096, groups of 128: 268 us (1184 TFLOP/s); of 64 with zero points 318 us
// (1001); of 32 469 us (678). 8192 tokens of 32 experts, top 4, 4096 x 1024: 907 us (909) one at a
// time, 1045 (789) one after the other, where the power limit lowers the clock.
// Every wait is bounded; one that runs out records PRISM_MOE_ERR_TIMEOUT and the CTA drains its
// copies and MMAs before it frees TMEM.
#include <algorithm>
#include <type_traits>

#include "gemm_sm100.cuh"
#include "internal.h"
#include "w4.cuh"

namespace prism {
namespace {

constexpr int kRowsW = 128;      // weight rows per tile
// Average rows per segment up to which tiles are narrow, for every group size. 128 experts of
// 2048 x 768, both products, narrow and wide, 32, 64 and 80 rows on average: groups of 128 195 and
// 289 us, 285 and 304, 369 and 311; of 64 with zero points 241 and 315, 356 and 358, 440 and 374; of 32
// 361 and 425, 534 and 580, 662 and 601; with zero points 377 and 406, 533 and 560, 709 and 580. One
// segment, 18944 x 4096, groups of 128: 64 rows 35.0 and 36.9 us, 96 rows 45 and 37.
constexpr int kNarrowRows = 64;
constexpr int kTokBox = 64;      // activation rows per copy
constexpr int kPackStage = 8 * 1024;
constexpr size_t kPrefixW4 = ((kMaxW4Segments + 1) * 4 + 15) / 16 * 16;

// The shapes: 256 activation rows (many rows per segment: one decoding serves them all) or 64 (tens of
// rows). With 64 a stage's work is shorter than the latency of handing it from role to role (about 500
// cycles each, waits and votes included), so two CTAs share an SM and take turns; where there are no
// more tiles than SMs, one CTA has the whole SM's shared memory for its rings instead (4096 x 4096: 128 rows
// 30.7 us deep and 34.7 wide, 256 rows 32.7 and 38.9; 18944 x 4096: 64 rows 32.8 deep and 34.8 narrow.
// Eight decoding warps there instead of four changed nothing).
enum { kWide, kNarrow, kDeep };
template <int kShape>
struct Shape {
  static constexpr bool k64 = kShape != kWide;
  static constexpr int kTok = k64 ? 64 : 256;            // activation rows per tile, at most
  static constexpr int kAStage = kRowsW * kBK * 2;
  static constexpr int kStage = kAStage + kTok * kBK * 2;
  static constexpr int kStages = kShape == kWide ? 4 : kShape == kNarrow ? 3 : 7;
  static constexpr int kPackStages = kShape == kDeep ? 5 : 3;
  static constexpr int kAccWarps = k64 ? 4 : 8;
  static constexpr int kThreads = 256 + 32 * kAccWarps;
  static constexpr int kCtas = kShape == kNarrow ? 2 : 1;   // per SM
  static constexpr int kBufs = k64 ? 4 : 2;              // TMEM buffers, one group each
  static constexpr uint32_t kTmem = kBufs * kTok;        // TMEM columns
  // registers of the control, decoding and accumulating warpgroups; their sum is the launch's at
  // most (wide 128 x 4, narrow 80 x 3, deep 168 x 3)
  static constexpr int kRegsControl = 32;
  static constexpr int kRegsDecode = kShape == kNarrow ? 64 : 72;
  static constexpr int kRegsAcc = kShape == kNarrow ? 144 : 200;
};
constexpr int kDecWarps = 4;

// Shared memory after the stages: packed slots, zero-point slots, scale slots, barriers, prefix.
template <int G, int kShape>
struct Smem {
  using P = Shape<kShape>;
  static constexpr int kPG = 128 / G;                 // groups per chunk
  static constexpr int kZeroSlot = kRowsW * kPG;      // bytes
  static constexpr int kScaleSlot = kRowsW * kPG * 2;
  static constexpr int kScaleSlots = kPG == 4 ? 4 : 8;
  static constexpr int kPacked = P::kStages * P::kStage;
  static constexpr int kZeros = kPacked + P::kPackStages * kPackStage;
  static constexpr int kScales = kZeros + P::kPackStages * kZeroSlot;
  static constexpr int kBars = kScales + kScaleSlots * kScaleSlot;
  static constexpr int kNumBars = 2 * (P::kStages + P::kPackStages + kScaleSlots + P::kBufs) + 1;
  static constexpr int kPrefix = kBars + (kNumBars * 8 + 8 + 15) / 16 * 16;
  static constexpr int kBytes = 1024 + kPrefix + static_cast<int>(kPrefixW4);
  static_assert(kBytes <= (kShape == kNarrow ? 115712 : 232448), "shared memory budget");
};

struct LargeParams {
  int chunks, tiles, tiles_n;   // 128-input chunks, row tiles, M tiles
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
template <int kBatches, int kPairs>
__device__ __forceinline__ void add_scaled(float2 (&acc)[kPairs], uint32_t taddr, float s) {
  const float2 s2 = make_float2(s, s);
  const uint64_t ss = *reinterpret_cast<const uint64_t*>(&s2);
  uint32_t v[2][2][16];   // the next batch is on its way while this one is added
  tmem_ld16(taddr, v[0][0]);
  tmem_ld16(taddr + 16, v[0][1]);
#pragma unroll
  for (int b = 0; b < kBatches; ++b) {
    tmem_wait_ld();
    if (b + 1 < kBatches) {
      tmem_ld16(taddr + b * 32 + 32, v[(b + 1) & 1][0]);
      tmem_ld16(taddr + b * 32 + 48, v[(b + 1) & 1][1]);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i)
      fma2(acc[b * 16 + i], v[b & 1][i >> 3][2 * (i & 7)], v[b & 1][i >> 3][2 * (i & 7) + 1], ss);
  }
}

// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok));
  return ok != 0;
}
// Barriers, copies and accesses by shared-memory address.
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {   // all lanes, one answer
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "vote.sync.all.pred p, p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, uint32_t abort,
                                         uint64_t limit_ns) {
  if (__builtin_expect(bar_try(bar, parity), 1)) return true;
  const uint64_t t0 = global_timer_ns();
  while (true) {
    if (bar_try(bar, parity)) return true;
    if (__any_sync(0xffffffffu, lds32(abort) != 0 || global_timer_ns() - t0 > limit_ns)) return false;
  }
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void bar_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
               : "memory");
}
__device__ __forceinline__ void copy_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0,
                                        int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void copy_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0,
                                        int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
      : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ void sts128(uint32_t addr, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z),
               "r"(v.w)
               : "memory");
}
// kBytes (1, 2, 4 or 8) at ``addr``, low bytes first.
template <int kBytes>
__device__ __forceinline__ uint2 lds_small(uint32_t addr) {
  uint2 v = make_uint2(0, 0);
  if constexpr (kBytes == 8)
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  else if constexpr (kBytes == 4)
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v.x) : "r"(addr) : "memory");
  else if constexpr (kBytes == 2)
    asm volatile("{\n\t.reg .u16 h;\n\tld.shared.u16 h, [%1];\n\tcvt.u32.u16 %0, h;\n\t}"
                 : "=r"(v.x)
                 : "r"(addr)
                 : "memory");
  else
    asm volatile("{\n\t.reg .u16 h;\n\tld.shared.u8 h, [%1];\n\tcvt.u32.u16 %0, h;\n\t}"
                 : "=r"(v.x)
                 : "r"(addr)
                 : "memory");
  return v;
}

struct Tile {
  int e, mt;            // matrix, M tile
  int row0;             // first activation row
  int rows, cols;       // valid activation rows; MMA N (a multiple of 16)
  int c0;               // first chunk: tiles that share activations start at different ones
  int64_t begin, end;   // before finish(): the segment's rows as the table has them
  int part, parts;      //                  this tile's part of them
};

// A tile is looked up one ahead: the loads are issued by look_up and used by finish.
__device__ __forceinline__ Tile look_up(const LargeParams& p, const int32_t* prefix, int item) {
  Tile t;
  const int unit = item / p.tiles_n;
  t.mt = item % p.tiles_n;
  const int sg = find_segment(prefix, p.nseg, unit);
  t.part = unit - prefix[sg];
  t.parts = prefix[sg + 1] - prefix[sg];
  t.begin = p.seg_offsets ? p.seg_offsets[sg] : 0;
  t.end = p.seg_offsets ? p.seg_offsets[sg + 1] : p.rows_cap;
  t.e = p.seg_expert ? p.seg_expert[sg] : (p.num_mats == 1 ? 0 : sg);
  return t;
}
__device__ __forceinline__ Tile finish(const LargeParams& p, Tile t) {
  const int begin = static_cast<int>(max(t.begin, static_cast<int64_t>(0)));
  const int end = static_cast<int>(min(t.end, p.rows_cap));
  // a segment's rows in equal parts, each a multiple of 16
  const int per = ((end - begin + t.parts - 1) / t.parts + 15) / 16 * 16;
  t.row0 = begin + t.part * per;
  t.rows = max(0, min(per, end - t.row0));
  t.cols = max(16, (t.rows + 15) / 16 * 16);
  t.c0 = static_cast<int>(static_cast<int64_t>(t.mt) * p.chunks / p.tiles_n);
  return t;
}

// Ring position: slot and phase.
template <int kSlots>
struct Ring {
  int slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next() {
    if (++slot == kSlots) {
      slot = 0;
      phase ^= 1;
    }
  }
};

template <int G, bool kZeros, bool kSwiGLU, int kShape>
__global__ void __launch_bounds__(Shape<kShape>::kThreads, Shape<kShape>::kCtas)
    w4_large_kernel(const __grid_constant__ CUtensorMap map_x,
                    const __grid_constant__ CUtensorMap map_q,
                    const __grid_constant__ CUtensorMap map_s,
                    const __grid_constant__ CUtensorMap map_z, const LargeParams p) {
  using P = Shape<kShape>;
  using S = Smem<G, kShape>;
  constexpr int PG = S::kPG;
  constexpr int kTok = P::kTok, kStage = P::kStage, kAStage = P::kAStage;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  int32_t* prefix = reinterpret_cast<int32_t*>(smem + S::kPrefix);
  const uint32_t base = smem_u32(smem);
  const uint32_t packed = base + S::kPacked, zeros = base + S::kZeros, scales = base + S::kScales;
  const uint32_t full = base + S::kBars, empty = full + 8 * P::kStages;
  const uint32_t pk_full = empty + 8 * P::kStages, pk_empty = pk_full + 8 * P::kPackStages;
  const uint32_t sc_full = pk_empty + 8 * P::kPackStages, sc_empty = sc_full + 8 * S::kScaleSlots;
  const uint32_t acc_full = sc_empty + 8 * S::kScaleSlots, acc_empty = acc_full + 8 * P::kBufs;
  const uint32_t drain = acc_empty + 8 * P::kBufs, abort = drain + 12;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + (drain - base) + 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + (abort - base));

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    auto init = [&](uint32_t bar, int n, int count) {
      for (int i = 0; i < n; ++i)
        mbar_init(reinterpret_cast<uint64_t*>(smem + (bar - base)) + i, count);
    };
    init(full, P::kStages, 1 + kDecWarps);   // the copies' arrival and the decoding warps
    init(empty, P::kStages, 1);
    init(pk_full, P::kPackStages, 1);
    init(pk_empty, P::kPackStages, kDecWarps);
    init(sc_full, S::kScaleSlots, 1);
    init(sc_empty, S::kScaleSlots, P::kAccWarps);
    init(acc_full, P::kBufs, 1);
    init(acc_empty, P::kBufs, P::kAccWarps);
    init(drain, 1, 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&map_x);
    tma_prefetch_desc(&map_q);
    tma_prefetch_desc(&map_s);
    if (kZeros) tma_prefetch_desc(&map_z);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, P::kTmem);
    tmem_relinquish();
  }
  if (warp == 2) build_row_blocks(p.seg_offsets, p.nseg, p.rows_cap, kTok, prefix, p.min_rows);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int total = prefix[p.nseg] * p.tiles_n;
  auto give_up = [&]() {
    *abort_flag = 1;
    record_device_error(p.err, PRISM_MOE_ERR_TIMEOUT);
  };
  // ``body(tile)`` for every tile of this CTA, false to stop; tiles whose segment names no expert are
  // left out by every role alike
  auto for_tiles = [&](auto body) {
    bool ok = true;
    Tile next;
    if (blockIdx.x < total) next = look_up(p, prefix, blockIdx.x);
    for (int item = blockIdx.x; ok && item < total;) {
      const Tile t = finish(p, next);
      item += gridDim.x;
      if (item < total) next = look_up(p, prefix, item);
      if (t.e >= 0 && t.e < p.num_mats && t.rows > 0)
        ok = body(t);
      else if (warp == 2 && lane == 0 && t.rows > 0)
        record_device_error(p.err, PRISM_MOE_ERR_ARG);
    }
    return ok;
  };
  auto next_chunk = [&](int c) { return c + 1 == p.chunks ? 0 : c + 1; };
  // every lane polls: one lane polling for all (and the divergence it brings) measured 15% slower
  auto wait = [&](uint32_t bar, uint32_t parity) {
    return bar_wait(bar, parity, abort, p.wait_ns);
  };

  if (warp < 4) {
    reg_dealloc<P::kRegsControl>();
    bool ok = true;
    if (warp == 0) {
      // ---------------------------------------------------------------- activation rows
      // the kernel for short segments may run beside this one
      launch_dependents();
      Ring<P::kStages> st;
      ok = for_tiles([&](const Tile& t) {
        const int boxes = (t.cols + kTokBox - 1) / kTokBox;
        for (int i = 0, c = t.c0; i < p.chunks; ++i, c = next_chunk(c))
#pragma unroll
          for (int half = 0; half < 2; ++half) {   // inputs past the last are read as zeros
            if (!wait(empty + 8 * st.slot, st.phase ^ 1)) return false;
            if (elect_one()) {
              bar_expect(full + 8 * st.slot, boxes * kTokBox * kBK * 2);
              const uint32_t b = base + st.slot * kStage + kAStage;
              for (int x = 0; x < boxes; ++x)
                copy_2d(b + x * kTokBox * kBK * 2, &map_x, full + 8 * st.slot, (2 * c + half) * kBK,
                        t.row0 + x * kTokBox);
            }
            __syncwarp();
            st.next();
          }
        return true;
      });
    } else if (warp == 1) {
      // ---------------------------------------------------------------- MMA issuer
      Ring<P::kStages> st;
      Ring<P::kBufs> buf;
      constexpr int kSteps = G == 32 ? 2 : 4;   // 16-input steps of a group within 64 inputs
      const uint64_t desc_a = smem_desc_sw128(base), desc_b = smem_desc_sw128(base + kAStage);
      ok = for_tiles([&](const Tile& t) {
        const uint32_t idesc = idesc_bf16_f32(kRowsW, t.cols);
        for (int i = 0, c = t.c0; i < p.chunks; ++i, c = next_chunk(c)) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            if (!wait(full + 8 * st.slot, st.phase)) return false;
            const uint32_t off = st.slot * (kStage >> 4);
#pragma unroll
            for (int k0 = 0; k0 < 4; k0 += kSteps) {
              // a new group starts: its buffer must have been read
              const bool first = G != 128 || half == 0, last = G != 128 || half == 1;
              if (first && !wait(acc_empty + 8 * buf.slot, buf.phase ^ 1)) return false;
              tc_fence_after();
              if (elect_one()) {
#pragma unroll
                for (int kk = k0; kk < k0 + kSteps; ++kk)
                  tc_mma_bf16(tmem_base + buf.slot * kTok, desc_a + off + kk * 2,
                              desc_b + off + kk * 2, idesc, first && kk == k0 ? 0u : 1u);
                if (last) bar_commit(acc_full + 8 * buf.slot);
                if (k0 + kSteps == 4) bar_commit(empty + 8 * st.slot);
              }
              __syncwarp();
              if (last) buf.next();
            }
            st.next();
          }
        }
        return true;
      });
      if (!ok && lane == 0) give_up();
      __syncwarp();
      if (*abort_flag) {
        if (elect_one()) bar_commit(drain);   // completes once every MMA issued above has finished
        __syncwarp();
        const uint64_t t0 = global_timer_ns();
        while (!bar_try(drain, 0) &&
               !__any_sync(0xffffffffu, global_timer_ns() - t0 > kDrainNs)) {
        }
      }
    } else if (warp == 2) {
      // ---------------------------------------------------------------- packed weights
      Ring<P::kPackStages> pk;
      ok = for_tiles([&](const Tile& t) {
        const int tile0 = t.e * p.tiles + t.mt * 8;
        for (int i = 0, c = t.c0; i < p.chunks; ++i, c = next_chunk(c), pk.next()) {
          if (!wait(pk_empty + 8 * pk.slot, pk.phase ^ 1)) return false;
          if (elect_one()) {
            const uint32_t bar = pk_full + 8 * pk.slot;
            bar_expect(bar, kPackStage + (kZeros ? S::kZeroSlot : 0));
            copy_3d(packed + pk.slot * kPackStage, &map_q, bar, 0, c, tile0);
            if constexpr (kZeros) copy_3d(zeros + pk.slot * S::kZeroSlot, &map_z, bar, 0, c, tile0);
          }
          __syncwarp();
        }
        return true;
      });
    } else {
      // ---------------------------------------------------------------- scales
      Ring<S::kScaleSlots> sc;
      ok = for_tiles([&](const Tile& t) {
        for (int i = 0, c = t.c0; i < p.chunks; ++i, c = next_chunk(c), sc.next()) {
          if (!wait(sc_empty + 8 * sc.slot, sc.phase ^ 1)) return false;
          if (elect_one()) {
            bar_expect(sc_full + 8 * sc.slot, S::kScaleSlot);
            copy_3d(scales + sc.slot * S::kScaleSlot, &map_s, sc_full + 8 * sc.slot, 0, c,
                    t.e * p.tiles + t.mt * 8);
          }
          __syncwarp();
        }
        return true;
      });
    }
    if (!ok && lane == 0) give_up();
  } else if (warp < 8) {
    // ------------------------------------------------------------------ decode
    reg_dealloc<P::kRegsDecode>();
    constexpr int kTiles = 8 / kDecWarps;   // row tiles per warp
    const int w = warp - 4, g = lane >> 2, tq = lane & 3;
    const bool odd = g & 1;
    Ring<P::kStages> st;
    Ring<P::kPackStages> pk;
    // this lane's row g of the warp's first row tile: packed bytes, zero points, place in the A tile
    const uint32_t from = packed + kTiles * w * 1024 + lane * 16;
    const uint32_t zfrom = zeros + (kTiles * w * 16 + g) * PG;
    const uint32_t to = base + kTiles * w * 2048 + g * 128;
    const uint32_t at0 = ((odd ? 4 : 0) + tq) ^ g, at1 = ((odd ? 0 : 4) + tq) ^ g;
    const bool ok = for_tiles([&](const Tile& t) {
      for (int i = 0, c = t.c0; i < p.chunks; ++i, c = next_chunk(c)) {
        if (!wait(pk_full + 8 * pk.slot, pk.phase)) return false;
        // rows g and g + 8 of this warp's row tiles
        uint32_t zr[2 * kTiles][PG];
        uint4 v[2 * kTiles];
#pragma unroll
        for (int r = 0; r < 2 * kTiles; ++r) {
          v[r] = lds128(from + pk.slot * kPackStage + r * 512);
          uint32_t z = 0x08080808u;
          if constexpr (kZeros) z = lds_small<PG>(zfrom + pk.slot * S::kZeroSlot + r * 8 * PG).x;
#pragma unroll
          for (int j = 0; j < PG; ++j)
            zr[r][j] = kZeros ? (((z >> (8 * j)) & 0xfu) * 0x00010001u) | 0x43004300u : 0x43084308u;
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (!wait(empty + 8 * st.slot, st.phase ^ 1)) return false;
          const uint32_t a = to + st.slot * kStage;
#pragma unroll
          for (int r = 0; r < 2 * kTiles; ++r) {
            // lanes of odd rows take the two words in the other order: their 16-byte stores then
            // fall into the other half of the banks
#pragma unroll
            for (int i2 = 0; i2 < 2; ++i2) {
              const uint32_t w0 = word_of(v[r], 2 * half + i2), w1 = word_of(v[r], 2 * half + 1 - i2);
              const uint32_t word = odd ? w1 : w0;
              uint32_t zero = zr[r][0];
              if constexpr (PG == 2) zero = zr[r][half];
              if constexpr (PG == 4) zero = odd ? zr[r][2 * half + 1 - i2] : zr[r][2 * half + i2];
              sts128(a + r * 1024 + ((i2 ? at1 : at0) << 4),
                     make_uint4(code_pair(word, 0, zero), code_pair(word, 1, zero),
                                code_pair(word, 2, zero), code_pair(word, 3, zero)));
            }
          }
          fence_async_smem();
          __syncwarp();
          if (lane == 0) bar_arrive(full + 8 * st.slot);
          st.next();
        }
        // given back once the stores above have used it: an arrival right after the loads can overtake
        // them, and the next copy then lands under a load in flight
        __syncwarp();
        if (lane == 0) bar_arrive(pk_empty + 8 * pk.slot);
        pk.next();
      }
      return true;
    });
    if (!ok && lane == 0) give_up();
  } else {
    // ------------------------------------------------------------------ accumulate
    reg_alloc<P::kRegsAcc>();
    const int q = warp & 3, side = (warp - 8) >> 2;   // narrow: one side, all columns
    constexpr int kPairs = P::k64 ? 32 : 64;          // pairs of columns held, at most
    Ring<P::kBufs> buf;
    Ring<S::kScaleSlots> sl;
    int held = -1;
    const int row = q * 32 + lane;                     // weight row in the tile
    const bool ok = for_tiles([&](const Tile& t) {
      const int left = P::k64 ? t.cols : (t.cols / 16 + 1) / 2 * 16;   // columns of side 0
      const int col0 = side ? left : 0, ncols = side ? t.cols - left : left;
      float2 acc[kPairs];
#pragma unroll
      for (int i = 0; i < kPairs; ++i) acc[i] = make_float2(0.f, 0.f);
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + col0;
      // every chunk of the tile, 32 kBatches columns of each group (those past ncols hold what an
      // earlier tile left there and are never stored)
      auto add_chunks = [&](auto batches) {
        constexpr int kBatches = decltype(batches)::value;
        for (int i = 0; i < p.chunks; ++i) {
          if (!wait(sc_full + 8 * sl.slot, sl.phase)) return false;
          const uint2 raw = lds_small<2 * PG>(scales + sl.slot * S::kScaleSlot + row * 2 * PG);
          const float sc[4] = {__uint_as_float(raw.x << 16), __uint_as_float(raw.x & 0xffff0000u),
                               __uint_as_float(raw.y << 16), __uint_as_float(raw.y & 0xffff0000u)};
          // the slot before this one is given back now, when its scales have been used for certain
          __syncwarp();
          if (lane == 0 && held >= 0) bar_arrive(sc_empty + 8 * held);
          held = sl.slot;
          sl.next();
#pragma unroll
          for (int gr = 0; gr < PG; ++gr) {
            if (!wait(acc_full + 8 * buf.slot, buf.phase)) return false;
            tc_fence_after();
            if constexpr (kBatches > 0) add_scaled<kBatches>(acc, taddr + buf.slot * kTok, sc[gr]);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(acc_empty + 8 * buf.slot);
            buf.next();
          }
        }
        return true;
      };
      bool done;
      switch ((ncols + 31) >> 5) {   // once per tile: a choice per group would copy the sums about
        case 0: done = add_chunks(std::integral_constant<int, 0>{}); break;
        case 1: done = add_chunks(std::integral_constant<int, 1>{}); break;
        case 2: done = add_chunks(std::integral_constant<int, 2>{}); break;
        case 3: done = add_chunks(std::integral_constant<int, P::k64 ? 2 : 3>{}); break;
        default: done = add_chunks(std::integral_constant<int, P::k64 ? 2 : 4>{}); break;
      }
      if (!done) return false;
      // ---- output: a lane is one output of every activation row, so 32 lanes store 64 bytes of a row
      // (16-byte stores after swapping columns between lanes took half as long again: the shuffles
      // cost more than the stores they save)
      const int64_t ld = p.n_out;
      if constexpr (kSwiGLU) {
        // lanes 0-7 and 16-23 hold gate rows, the lanes 8 above them the matching up rows; of two
        // columns the gate lane finishes the first, the up lane the second
        const bool up = lane & 8;
        const int n = (t.mt * kRowsW + q * 32) / 2 + (lane >> 4) * 8 + (lane & 7);
        const int mine = col0 + (up ? 1 : 0);
        uint16_t* to = p.out + (t.row0 + mine) * ld + n;
        const int rows = n < p.n_out ? min(t.rows, col0 + ncols) - mine : 0;
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
          const float got = __shfl_xor_sync(0xffffffffu, up ? acc[i].x : acc[i].y, 8);
          const float h = silu_mul(up ? got : acc[i].x, up ? acc[i].y : got);
          if (2 * i < rows) *to = float_to_bf16_bits(h);
          to += 2 * ld;
        }
      } else {
        const int n = t.mt * kRowsW + row;
        uint16_t* to = p.out + (t.row0 + col0) * ld + n;
        const int rows = n < p.n_out ? min(ncols, t.rows - col0) : 0;
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
          const uint32_t d = cvt_bf16x2(acc[i].x, acc[i].y);
          if (2 * i < rows) to[0] = static_cast<uint16_t>(d);
          if (2 * i + 1 < rows) to[ld] = static_cast<uint16_t>(d >> 16);
          to += 2 * ld;
        }
      }
      return true;
    });
    if (!ok && lane == 0) give_up();
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    // copies that a given-up wait left in flight land within microseconds: give them a millisecond
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 1000000ull) {
    }
  }
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, P::kTmem);
  }
}

struct Maps {
  CUtensorMap x, q, s, z;
};

template <int G, bool kZeros, bool kSwiGLU, int kShape>
int launch_shape(const Maps& map, const LargeParams& p, int grid, cudaStream_t st) {
  auto kern = w4_large_kernel<G, kZeros, kSwiGLU, kShape>;
  if (int r = ensure_smem_attr(reinterpret_cast<const void*>(kern), Smem<G, kShape>::kBytes))
    return r;
  // a plain launch, after the end of the kernel before it: started while gate_up ended, the down product
  // of a skewed batch (4096 tokens of 128 experts) made both 690 us instead of 620
  kern<<<grid, Shape<kShape>::kThreads, Smem<G, kShape>::kBytes, st>>>(map.x, map.q, map.s, map.z, p);
  PRISM_LAUNCH_CHECK("w4_large_kernel launch");
  return PRISM_MOE_OK;
}

template <int G, bool kZeros, bool kSwiGLU>
int launch_large(const Maps& map, const LargeParams& p, int shape, int grid, cudaStream_t st) {
  if (shape == kDeep) return launch_shape<G, kZeros, kSwiGLU, kDeep>(map, p, grid, st);
  return shape == kNarrow ? launch_shape<G, kZeros, kSwiGLU, kNarrow>(map, p, grid, st)
                          : launch_shape<G, kZeros, kSwiGLU, kWide>(map, p, grid, st);
}

template <int G>
int launch_group(const Maps& map, const LargeParams& p, bool swiglu, int shape, int grid,
                 cudaStream_t st) {
  if (p.z)
    return swiglu ? launch_large<G, true, true>(map, p, shape, grid, st)
                  : launch_large<G, true, false>(map, p, shape, grid, st);
  return swiglu ? launch_large<G, false, true>(map, p, shape, grid, st)
                : launch_large<G, false, false>(map, p, shape, grid, st);
}

}  // namespace

int w4_product_large(const W4Problem& pr, int min_rows, cudaStream_t st) {
  LargeParams p{};
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
  const int64_t stack = static_cast<int64_t>(p.tiles) * pr.num_mats;   // row tiles of all matrices
  PRISM_CHECK_ARG(stack < (int64_t(1) << 31), "4-bit product: too many weight rows");
  Maps map;
  {
    const uint64_t dims[2] = {static_cast<uint64_t>(pr.K), static_cast<uint64_t>(pr.rows_cap)};
    const uint64_t strides[1] = {static_cast<uint64_t>(pr.K) * 2};
    const uint32_t box[2] = {kBK, kTokBox};
    if (int r = encode_bf16_map(&map.x, pr.x, 2, dims, strides, box)) return r;
  }
  // per chunk and 8 row tiles: 1 KB of codes, 16 rows' scales and zero points of each
  auto tiles_map = [&](CUtensorMap* m, CUtensorMapDataType type, const void* at, int elems, int bytes) {
    const uint64_t dims[3] = {static_cast<uint64_t>(elems), static_cast<uint64_t>(p.chunks),
                              static_cast<uint64_t>(stack)};
    const uint64_t strides[2] = {static_cast<uint64_t>(bytes),
                                 static_cast<uint64_t>(bytes) * p.chunks};
    const uint32_t box[3] = {static_cast<uint32_t>(elems), 1, 8};
    return encode_map(m, type, CU_TENSOR_MAP_SWIZZLE_NONE, at, 3, dims, strides, box);
  };
  const int pg = 128 / pr.w.group_size;
  if (int r = tiles_map(&map.q, CU_TENSOR_MAP_DATA_TYPE_UINT32, p.q, 256, 1024)) return r;
  if (int r = tiles_map(&map.s, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, p.s, 16 * pg, 32 * pg)) return r;
  map.z = map.s;
  if (p.z)
    if (int r = tiles_map(&map.z, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.z, 16 * pg, 16 * pg)) return r;
  const int64_t long_segs = std::min<int64_t>(pr.nseg, pr.rows_cap / (min_rows + 1));
  // most tiles there can be, of 64 rows or of 256
  auto tiles_of = [&](int rows) {
    return (pr.seg_offsets ? pr.rows_cap / rows + long_segs : ceil_div(pr.rows_cap, rows)) * p.tiles_n;
  };
  const int sms = num_sms();
  const int shape = tiles_of(64) <= sms                                                ? kDeep
                    : pr.rows_cap <= kNarrowRows * static_cast<int64_t>(pr.nseg) ? kNarrow
                                                                                 : kWide;
  const int64_t items = tiles_of(shape == kWide ? 256 : 64);
  PRISM_CHECK_ARG(items < (int64_t(1) << 31), "4-bit product: too many tiles");
  const int grid = static_cast<int>(
      std::max<int64_t>(1, std::min<int64_t>(items, sms * (shape == kNarrow ? 2 : 1))));
  switch (pr.w.group_size) {
    case 32: return launch_group<32>(map, p, pr.swiglu, shape, grid, st);
    case 64: return launch_group<64>(map, p, pr.swiglu, shape, grid, st);
    default: return launch_group<128>(map, p, pr.swiglu, shape, grid, st);
  }
}

}  // namespace prism
