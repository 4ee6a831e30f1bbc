// Products with 4-bit weights for few rows: y[r, n] = sum_k x[r, k] * (code[n, k] - zero) * scale.
//
// Weights come in tiles of 16 rows by 128 inputs, 1 KB each (w4.cuh). One warp-wide pair of 16-byte
// loads brings a tile: lane 4 g + t holds 32 codes of row g and 32 of row g + 8, four words of 8
// consecutive inputs each. The products run on the m16n8k16 tensor instruction with the weights as
// its 16 rows and 8 activation rows as its columns: a lane's word gives the A fragments of two
// instructions without any exchange (the order of the inputs inside one sum is free, as long as both
// operands agree), and the B fragments are x itself, one 16-byte load per word.
//
// Codes become bf16 by bits: 0x4300 | code is 128 + code, exactly; subtracting 128 + zero leaves the
// signed integer, exactly. The instruction multiplies integers by activations and sums in fp32; the
// scale is applied to the fp32 sum of each group, so no weight is ever rounded.
//
// The subtraction of 128 + zero that code_pair does would be a third of the decoding. It is left out
// here: the instruction sums (offset + code) * x, and offset * x and zero * x of the group are taken
// off together with the scale; those sums come from one or two more instructions per input step, on
// constant matrices, once per block of rows. The offset is 128 where the nibble is used in place and
// 16 where one bit's shift puts it under a smaller exponent (w4.cuh), which makes three shifts per
// word: shifts and logic share a half-rate pipe and are what the loop has most of. The price is
// cancellation: the sums carry up to 143 per input instead of 8, at most 2^-17 of their terms'
// magnitudes at 4096 inputs where the output's rounding is 2^-8; and range: 143 * 128 * |x| stays in
// fp32 up to |x| = 2^113.
//
// What bounds it: few rows reuse nothing, so every hit weight crosses HBM once and that is the floor.
// What keeps it from that is latency inside the warps: 16 of them an SM, as many as registers allow, each
// with copy, wait, decoding, product and sum in line (counters of the decode call below: HBM 46%, SM 48%
// busy). More warps with fewer registers (24 of 80) spilled and took 10% longer, smaller and deeper
// steps as well. Measured: 1 x 18944 x 4096 17.0 us (2.3 TB/s of codes), 16 rows 24.6; 64 tokens of 128
// experts, top 8, 2048 x 768, both products 88 us (3.5 TB/s); one token of them 17, where two
// launches and three memory latencies are most of it.
// A block's warps split the inputs (kw ways) and keep their part of x in registers while the block
// streams its row tiles (up to 2048 inputs; of longer rows every item loads x again, part by part); the
// partial sums meet in shared memory in a fixed order. Every lane copies the 16-byte pieces that it will
// use itself (cp.async, kDepth row tiles ahead, across the borders of blocks of rows), so no barrier
// stands between a copy and its use. Blocks take equal runs of a device-side list of (segment's rows,
// output tiles), so the host needs no counts.
#include <algorithm>

#include "internal.h"
#include "segments.cuh"
#include "w4.cuh"

namespace prism {
namespace {

constexpr int kWarps = 8;
constexpr int kSmallRows = 16;
constexpr int kCh = 2;          // 128-input chunks a warp keeps in registers per pass
constexpr int kDepth = 2;       // steps in flight per warp, the one in use included
constexpr int kMaxKwRt = 4;     // kw * rt <= kWarps * kMaxKwRt
constexpr int kTps = 2;         // row tiles per step
constexpr int kMaxRt = 4;       // row tiles per item
constexpr int kColStride = 20;  // floats between the columns of a partial tile: no bank conflicts

// How a launch follows the kernel before it: after its end; early (it may start while that one ends,
// and waits before it reads what that one wrote); beside it (it reads nothing that one writes, and
// only ends after it).
enum { kAfter, kEarly, kBeside };

struct SmallParams {
  const uint16_t* x;
  int64_t ld_x;              // elements; = inputs
  int K, chunks;             // inputs, ceil(inputs / 128)
  int tiles;                 // 16-row tiles of one matrix
  int n_out;                 // columns of ``out`` (gate_up: inter)
  uint16_t* out;
  int64_t rows_cap;
  const int32_t* seg_offsets;   // NULL: one segment [0, rows_cap)
  const int32_t* seg_expert;
  int nseg, num_mats;
  const uint8_t *q, *z;
  const uint16_t* s;
  int kw, rw, rt, passes;    // input splits, row-tile splits, row tiles per item, input passes
  int rt_bits;               // rt = 1 << rt_bits
  int blocks_n;              // ceil(tiles / rt)
  int all_chunks;            // of all matrices
  int64_t max_rows;          // longer segments are the other kernel's
  int start;                 // kAfter, kEarly or kBeside
  int* err;
};

__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                          uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int B>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
  if constexpr (B == 16)
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(dst), "l"(src));
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(B));
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Scales and zero points of one chunk of a row tile, 4 lanes to a row g: lane t = 0 and 1 copy the
// scales of rows g and g + 8, t = 2 and 3 the zero points, in pieces of kMetaBytes (which hold
// neighbouring rows too where a row has fewer bytes than a copy must have).
template <int PG>
struct Meta {
  static constexpr int kBytes = PG == 4 ? 8 : 4;
  static constexpr int kScaleRows = PG == 1 ? 2 : 1;                // rows in a piece of scales
  static constexpr int kZeroRows = PG == 4 ? 2 : PG == 2 ? 2 : 4;   // rows in a piece of zero points
};

template <int G, bool kZeros, bool kSwiGLU, int NT>
__global__ void __launch_bounds__(32 * kWarps, NT == 1 ? 2 : 1) w4_small_kernel(const SmallParams p) {
  constexpr int PG = 128 / G;   // groups per chunk
  using M = Meta<PG>;
  // mixed offsets keep two sums per group; with four groups a chunk that is more registers than the
  // shift is worth, and the offset is 16 for every nibble
  constexpr bool kMixed = PG < 4;
  constexpr bool kOff = kMixed || !kZeros;
  constexpr int kMetaSlot = 32 * M::kBytes;
  constexpr int kSlot = kTps * kCh * (1024 + kMetaSlot);
  extern __shared__ uint4 smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(smem_raw);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int nwarps = blockDim.x >> 5;
  uint8_t* ring = smem + warp * kDepth * kSlot;
  const uint32_t ring_at = smem_u32(ring);
  float* part = reinterpret_cast<float*>(smem + nwarps * kDepth * kSlot);
  const int g = lane >> 2, t = lane & 3;
  const int wk = warp % p.kw, wr = warp / p.kw;
  constexpr int kTile = 8 * NT * kColStride;          // floats of a partial tile
  int32_t* prefix = reinterpret_cast<int32_t*>(part + 2 * p.kw * p.rt * kTile);

  build_row_blocks_cta(p.seg_offsets, p.nseg, p.rows_cap, 8 * NT, prefix, p.max_rows);
  const int total = prefix[p.nseg] * p.blocks_n;
  // this block's run of items
  const int64_t bid = blockIdx.x, blocks = gridDim.x;
  const int item0 = static_cast<int>(total * bid / blocks);
  const int item1 = static_cast<int>(total * (bid + 1) / blocks);
  // a grid that ended before the one ahead of it would let the next one pass both
  const bool hold = p.start == kEarly || blockIdx.x == 0;
  if (item0 >= item1) {
    if (hold) wait_for_earlier();
    return;
  }

  // ---- the stream of steps: item by item, pass by pass, kTps row tiles a step. Every item has the
  // same steps and every step the same copies: what lies past the last tile or chunk is read from
  // the last one instead and its sums are not used (or its x is zero).
  struct Place {
    int unit, nb, base;   // unit's rows, item of the unit, first row tile of its matrix (< 0: none)
  };
  auto matrix = [&](int unit) {
    const int sg = find_segment(prefix, p.nseg, unit);
    const int e = p.seg_expert ? p.seg_expert[sg] : (p.num_mats == 1 ? 0 : sg);
    return e >= 0 && e < p.num_mats ? e * p.tiles : -1;
  };
  auto step_on = [&](Place& at, bool more) {
    if (++at.nb == p.blocks_n) {
      at.nb = 0;
      ++at.unit;
      if (more) at.base = matrix(at.unit);
    }
  };
  const int first_i = wr * kTps, next_i = p.rw * kTps;
  // this lane's pieces: 16 bytes of rows g and g + 8, and scales (t < 2) or zero points
  const int meta_row = g + 8 * (t & 1);
  const uint8_t* q_lane = p.q + lane * 16;
  const uint8_t* m_lane =
      t < 2 ? reinterpret_cast<const uint8_t*>(p.s) + (meta_row & ~(M::kScaleRows - 1)) * PG * 2
            : p.z + (meta_row & ~(M::kZeroRows - 1)) * PG;
  const int m_stride = t < 2 ? 32 * PG : 16 * PG;
  const uint32_t ring_lane = ring_at + lane * 16, ring_meta = ring_at + lane * M::kBytes;
  Place ahead{item0 / p.blocks_n, item0 % p.blocks_n, 0};
  ahead.base = matrix(ahead.unit);
  Place now = ahead;
  int ahead_item = item0, ahead_pass = 0, ahead_i = first_i;
  uint32_t fill = 0, use = 0;   // byte offsets of the slots
  auto fetch = [&]() {
    if (ahead_item < item1) {
      const int c0 = (ahead_pass * p.kw + wk) * kCh;
      const int tile0 = ahead.nb * p.rt + ahead_i;
      const int chunk0 = (max(ahead.base, 0) + tile0) * p.chunks + c0;
      // tiles and chunks past the end of a row of tiles are the next ones' in memory: only the end of
      // the whole stack needs care
      const bool inside = chunk0 + (kTps - 1) * p.chunks + kCh <= p.all_chunks;
#pragma unroll
      for (int u = 0; u < kTps; ++u) {
        int chunk = chunk0 + u * p.chunks;
        const uint8_t* from = q_lane + static_cast<int64_t>(chunk) * 1024;
        const uint8_t* meta = m_lane + static_cast<int64_t>(chunk) * m_stride;
#pragma unroll
        for (int ch = 0; ch < kCh; ++ch) {
          if (!inside) {
            chunk = min(chunk0 + u * p.chunks + ch, p.all_chunks - 1);
            from = q_lane + static_cast<int64_t>(chunk) * 1024;
            meta = m_lane + static_cast<int64_t>(chunk) * m_stride;
          }
          const uint32_t to = ring_lane + fill + (u * kCh + ch) * (1024 + kMetaSlot);
          copy_async<16>(to, from);
          copy_async<16>(to + 512, from + 512);
          if (kZeros || t < 2)
            copy_async<M::kBytes>(ring_meta + fill + (u * kCh + ch) * (1024 + kMetaSlot) + 1024, meta);
          from += 1024;
          meta += m_stride;
        }
      }
      ahead_i += next_i;
      if (ahead_i >= p.rt) {
        ahead_i = first_i;
        if (++ahead_pass == p.passes) {
          ahead_pass = 0;
          ++ahead_item;
          step_on(ahead, ahead_item < item1);
        }
      }
    }
    copy_commit();
    fill = fill == (kDepth - 1) * kSlot ? 0 : fill + kSlot;
  };
#pragma unroll
  for (int d = 0; d < kDepth - 1; ++d) fetch();

  // From here on this kernel reads what the one before it wrote. Everything above (the list, the
  // weights in flight) may run while that one ends; a kernel behind may start likewise.
  launch_dependents();
  if (p.start != kBeside) wait_for_earlier();
  uint4 xb[kCh][NT][4];
  // sums over each group, columns 2 t and 2 t + 1: of offset * x (with zero point 8 where there are
  // none), and of x
  float off[kOff ? kCh : 1][PG][NT][2], sx[kZeros ? kCh : 1][PG][NT][2];
  int loaded_unit = -1, loaded_pass = -1;
  int rows = 0;
  int64_t row0 = 0;
  for (int item = item0, round = 0; item < item1; ++item, round ^= 1) {
    if (now.unit != loaded_unit) {
      const int sg = find_segment(prefix, p.nseg, now.unit);
      const RowSpan span = segment_rows(p.seg_offsets, sg, p.rows_cap);
      row0 = span.begin + static_cast<int64_t>(now.unit - prefix[sg]) * 8 * NT;
      rows = static_cast<int>(min(static_cast<int64_t>(8 * NT), span.end - row0));
    }
    float* sums = part + round * p.kw * p.rt * kTile;
    float* mine = sums + wk * p.rt * kTile + 2 * t * kColStride + g;
    for (int pass = 0; pass < p.passes; ++pass) {
      if (now.unit != loaded_unit || pass != loaded_pass) {
        // this warp's part of x: rows g (+ 8 nt), inputs 8 t .. 8 t + 7 of each 32
        const int c0 = (pass * p.kw + wk) * kCh;
        loaded_unit = now.unit;
        loaded_pass = pass;
#pragma unroll
        for (int c = 0; c < kCh; ++c)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int k = (c0 + c) * 128 + j * 32 + t * 8;
              const bool ok = g + 8 * nt < rows && k < p.K;
              xb[c][nt][j] =
                  ok ? *reinterpret_cast<const uint4*>(p.x + (row0 + g + 8 * nt) * p.ld_x + k)
                     : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
        for (int c = 0; c < kCh; ++c)
#pragma unroll
          for (int gr = 0; gr < PG; ++gr)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              float o[4] = {}, ones[4] = {};
              constexpr uint32_t one = 0x3f803f80u;                      // 1
              constexpr uint32_t at_0 = !kMixed ? (kZeros ? 0x41804180u : 0x41c041c0u)
                                                : (kZeros ? 0x43004300u : 0x43084308u);   // 128 (+ 8)
              constexpr uint32_t at_1 = kZeros ? 0x41804180u : 0x41c041c0u;   // 16 (+ 8)
#pragma unroll
              for (int j = gr * (4 / PG); j < (gr + 1) * (4 / PG); ++j) {
                if constexpr (kOff) {
                  mma_16816(o, at_0, at_0, at_1, at_1, xb[c][nt][j].x, xb[c][nt][j].y);
                  mma_16816(o, at_0, at_0, at_1, at_1, xb[c][nt][j].z, xb[c][nt][j].w);
                }
                if constexpr (kZeros) {
                  mma_16816(ones, one, one, one, one, xb[c][nt][j].x, xb[c][nt][j].y);
                  mma_16816(ones, one, one, one, one, xb[c][nt][j].z, xb[c][nt][j].w);
                }
              }
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                if constexpr (kOff) off[c][gr][nt][q] = o[q];
                if constexpr (kZeros) sx[c][gr][nt][q] = ones[q];
              }
            }
      }
#pragma unroll 1
      for (int i0 = first_i; i0 < p.rt; i0 += next_i) {
        __syncwarp();   // every lane has read the slot that the next copies fill
        fetch();
        copy_wait<kDepth - 1>();
        __syncwarp();   // scales and zero points were copied by other lanes of the row
        const uint8_t* slot = ring + use;
        use = use == (kDepth - 1) * kSlot ? 0 : use + kSlot;
#pragma unroll
        for (int u = 0; u < kTps; ++u) {
          float acc[NT][4] = {};
#pragma unroll
          for (int c = 0; c < kCh; ++c) {
            const uint8_t* at = slot + (u * kCh + c) * (1024 + kMetaSlot);
            const uint4 w0 = *reinterpret_cast<const uint4*>(at + lane * 16);
            const uint4 w1 = *reinterpret_cast<const uint4*>(at + lane * 16 + 512);
            const uint8_t* meta = at + 1024 + g * 4 * M::kBytes;
            float sc[2][PG], zp[2][PG];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              load_scales<PG>(reinterpret_cast<const uint16_t*>(meta + h * M::kBytes) +
                                  (g & (M::kScaleRows - 1)) * PG,
                              sc[h]);
              if constexpr (kZeros)
                load_zero_points<PG>(meta + (2 + h) * M::kBytes + (g & (M::kZeroRows - 1)) * PG, zp[h]);
            }
#pragma unroll
            for (int gr = 0; gr < PG; ++gr) {
              float sum[NT][4] = {};
#pragma unroll
              for (int j = gr * (4 / PG); j < (gr + 1) * (4 / PG); ++j) {
                const uint32_t word0 = word_of(w0, j), word1 = word_of(w1, j);
                uint32_t a[2][4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                  a[0][q] = offset_pair<kMixed>(word0, q);
                  a[1][q] = offset_pair<kMixed>(word1, q);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                  mma_16816(sum[nt], a[0][0], a[1][0], a[0][1], a[1][1], xb[c][nt][j].x,
                            xb[c][nt][j].y);
                  mma_16816(sum[nt], a[0][2], a[1][2], a[0][3], a[1][3], xb[c][nt][j].z,
                            xb[c][nt][j].w);
                }
              }
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                  float d = sum[nt][q];
                  if constexpr (kOff) d -= off[c][gr][nt][q & 1];
                  if constexpr (kZeros)
                    d = fmaf(kMixed ? -zp[q >> 1][gr] : -16.f - zp[q >> 1][gr],
                             sx[c][gr][nt][q & 1], d);
                  acc[nt][q] = fmaf(sc[q >> 1][gr], d, acc[nt][q]);
                }
            }
          }
          float* to = mine + (i0 + u) * kTile;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              float* v = to + (8 * nt + (q & 1)) * kColStride + 8 * (q >> 1);
              *v = pass == 0 ? acc[nt][q] : *v + acc[nt][q];   // the same lane's own sum
            }
        }
      }
    }
    // one barrier per item: partial sums have two buffers, and a warp cannot be two items ahead
    __syncthreads();
    const int nb = now.nb, base = now.base, tiles_here = min(p.tiles - nb * p.rt, p.rt);
    step_on(now, item + 1 < item1);
    if (base < 0) {   // an id no weights belong to: recorded, nothing written
      if (threadIdx.x == 0) record_device_error(p.err, PRISM_MOE_ERR_ARG);
      continue;
    }
    // sum of the kw partial tiles, two outputs per thread, neighbours along the output row
    constexpr int kPairs = kSwiGLU ? 4 : 8;   // output pairs of one row tile
    const int span_bits = p.rt_bits + (kSwiGLU ? 2 : 3);   // pairs of an item's output row
    for (int i = threadIdx.x; i < rows << span_bits; i += nwarps * 32) {
      const int col = i >> span_bits, pr = i & ((1 << span_bits) - 1);
      const int tile = pr / kPairs, r = pr % kPairs * 2;
      if (tile >= tiles_here) continue;
      const float* at = sums + tile * kTile + col * kColStride + r;
      float2 a = make_float2(0.f, 0.f), b = make_float2(0.f, 0.f);
      for (int k = 0; k < p.kw; ++k, at += p.rt * kTile) {
        const float2 v = *reinterpret_cast<const float2*>(at);
        a.x += v.x;
        a.y += v.y;
        if constexpr (kSwiGLU) {
          const float2 u = *reinterpret_cast<const float2*>(at + 8);
          b.x += u.x;
          b.y += u.y;
        }
      }
      if constexpr (kSwiGLU) {
        a.x = silu_mul(a.x, b.x);
        a.y = silu_mul(a.y, b.y);
      }
      const int n = (nb * p.rt + tile) * 2 * kPairs + r;
      if (n < p.n_out)
        *reinterpret_cast<uint32_t*>(p.out + (row0 + col) * p.n_out + n) = pack_bf16x2(a.x, a.y);
    }
  }
  copy_wait<0>();
  if (p.start == kBeside && hold) wait_for_earlier();
}

template <int G, bool kZeros, bool kSwiGLU, int NT>
int launch_small(SmallParams p, int64_t units, cudaStream_t st) {
  auto kern = w4_small_kernel<G, kZeros, kSwiGLU, NT>;
  // inputs: up to 8 warps x 2 chunks per pass; warps that the inputs do not need take row tiles
  p.passes = static_cast<int>(ceil_div(p.chunks, kWarps * kCh));
  p.kw = static_cast<int>(ceil_div(p.chunks, p.passes * kCh));
  p.rw = 1;   // a power of two, and so are the row tiles of an item
  while (2 * p.rw * p.kw <= kWarps) p.rw *= 2;
  const int sms = num_sms();
  // row tiles per item and step: several share a barrier and the bookkeeping, few fill the GPU when
  // the call is small
  p.rt = p.rw * kTps;
  while (p.rt * 2 <= kMaxRt && units * ceil_div(p.tiles, p.rt * 2) >= 2 * sms) p.rt *= 2;
  constexpr int kSlot = kTps * kCh * (1024 + 32 * Meta<128 / G>::kBytes);
  constexpr int kTile = 8 * NT * kColStride;
  constexpr int kSmSmem = 233472;   // of one SM, 1 KB of it reserved per block
  const int warps = p.kw * p.rw;
  auto bytes_of = [&](int rt) {
    return warps * kDepth * kSlot + 2 * p.kw * rt * kTile * 4 + (p.nseg + 4) / 4 * 16;
  };
  // two blocks per SM where shorter items allow it
  if (NT == 1 && 2 * (bytes_of(p.rt) + 1024) > kSmSmem && p.rt >= 2 * kTps * p.rw) p.rt /= 2;
  const int bytes = bytes_of(p.rt);
  p.blocks_n = static_cast<int>(ceil_div(p.tiles, p.rt));
  p.rt_bits = 0;
  while ((1 << p.rt_bits) < p.rt) ++p.rt_bits;
  const int64_t all_chunks = static_cast<int64_t>(p.tiles) * p.num_mats * p.chunks;
  PRISM_CHECK_ARG(all_chunks < (int64_t(1) << 31) - 64, "4-bit product: too many weights");
  p.all_chunks = static_cast<int>(all_chunks);
  constexpr int kMaxBytes = kWarps * kDepth * kSlot + 2 * kWarps * kMaxKwRt * kTile * 4 +
                            (kMaxW4Segments + 4) / 4 * 16;
  static_assert(kMaxBytes <= 232448, "shared memory budget");
  if (int r = ensure_smem_attr(reinterpret_cast<const void*>(kern), kMaxBytes)) return r;
  const int64_t items = units * p.blocks_n;
  PRISM_CHECK_ARG(items < (int64_t(1) << 31), "4-bit product: too many outputs");
  const int per_sm = std::max(
      1, std::min({65536 / ((NT == 1 ? 128 : 256) * 32 * warps), kSmSmem / (bytes + 1024), 4}));
  const int grid =
      static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(items, per_sm * sms)));
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(32 * warps, 1, 1);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.start != kAfter ? 1 : 0;
  PRISM_CUDA(cudaLaunchKernelEx(&cfg, kern, p));
  return PRISM_MOE_OK;
}

template <int G, bool kZeros, bool kSwiGLU>
int launch_rows(const SmallParams& p, int64_t units8, int64_t units16, cudaStream_t st) {
  // 8 rows at a time (two blocks share an SM) while most segments have few more, else 16: a second pass
  // over the weights comes from L2 but is decoded again, so the limit is lower where a tile has more
  // scales and zero points. 128 experts of 2048 x 768, both products, 8 and 16 at a time: groups
  // of 128, 6 rows on average 103 and 156 us, 9 rows 137 and 162, 10 rows 146 and 162; of 64 without
  // zero points 9 rows 144 and 152, 10 rows 152 and 150; with zero points 7 rows 152 and 154, 8 rows 164
  // and 156; of 32, 6 rows 144 and 156, 7 rows 162 and 156. (8 experts of 4096 x 1024 turn at 7 rows.)
  // One segment of 8 rows, 18944 x 4096: 20.5 and 22.5; of 9: 28.7 and 22.5.
  constexpr int kRows = G == 128 || (G == 64 && !kZeros) ? 9 : 7;
  if (p.rows_cap > (p.seg_offsets ? kRows * static_cast<int64_t>(p.nseg) : 8))
    return launch_small<G, kZeros, kSwiGLU, 2>(p, units16, st);
  return launch_small<G, kZeros, kSwiGLU, 1>(p, units8, st);
}

template <int G, bool kZeros>
int launch_mode(const SmallParams& p, bool swiglu, int64_t u8, int64_t u16, cudaStream_t st) {
  return swiglu ? launch_rows<G, kZeros, true>(p, u8, u16, st)
                : launch_rows<G, kZeros, false>(p, u8, u16, st);
}

template <int G>
int launch_zeros(const SmallParams& p, bool swiglu, int64_t u8, int64_t u16, cudaStream_t st) {
  return p.z ? launch_mode<G, true>(p, swiglu, u8, u16, st)
             : launch_mode<G, false>(p, swiglu, u8, u16, st);
}

}  // namespace

int w4_product(const W4Problem& pr, cudaStream_t st) {
  SmallParams p{};
  p.max_rows = int64_t(1) << 31;
  // Few rows: this kernel alone (a longer segment runs in blocks of 16 rows, its weights from L2
  // after the first). Without a table: up to 16 rows, and up to 64 while the matrix is so small that
  // the other kernel's tiles could not fill the GPU (17 x 4096 x 4096: 17 us here, 29 there;
  // 17 x 18944 x 4096: 39 and 33). With one: segments of 12 rows on average, for every group size
  // (128 experts of 2048 x 768, both products, here and with both kernels, 12 and 16 rows on average:
  // groups of 128 169 and 189 us, 222 and 175; of 64 with zero points 167 and 184, 214 and 194; of 32
  // 174 and 188, 223 and 213; with zero points 186 and 200, 239 and 222). Else segments of at most
  // kSmallRows rows run here and longer ones on the other kernel; the host does not know the lengths
  // and launches both.
  // the lists of row blocks and output tiles count in 32 bits
  PRISM_CHECK_ARG(ceil_div(pr.rows_cap, 8) * pr.nseg < (int64_t(1) << 31), "4-bit product: too many rows");
  const int64_t out_tiles = ceil_div(pr.swiglu ? 2 * pr.n_out : pr.n_out, 16);
  const bool few = pr.seg_offsets
                       ? pr.rows_cap <= std::max<int64_t>(kSmallRows, 12 * pr.nseg)
                       : pr.rows_cap <= kSmallRows ||
                             (pr.rows_cap <= 64 && ceil_div(pr.rows_cap, 16) * out_tiles <= 9 * num_sms());
  if (!few) {
    if (int r = w4_product_large(pr, kSmallRows, st)) return r;
    if (!pr.seg_offsets) return PRISM_MOE_OK;
    p.max_rows = kSmallRows;
  }
  // The two kernels of a product share neither rows nor weights, so this one fills the SMs that the
  // other's last tiles leave (333 tokens of 60 experts, top 4, 1440 x 736, groups of 32 with zero points,
  // both products: 96 us, one kernel after the other 107; 4096 tokens of 128 experts, skewed: 607
  // and 634).
  p.start = !few ? kBeside : pr.after_product ? kEarly : kAfter;
  p.x = static_cast<const uint16_t*>(pr.x);
  p.ld_x = pr.K;
  p.K = static_cast<int>(pr.K);
  p.chunks = static_cast<int>(ceil_div(pr.K, 128));
  p.tiles = static_cast<int>(ceil_div(pr.swiglu ? 2 * pr.n_out : pr.n_out, 16));
  p.n_out = static_cast<int>(pr.n_out);
  p.out = static_cast<uint16_t*>(pr.out);
  p.rows_cap = pr.rows_cap;
  p.seg_offsets = pr.seg_offsets;
  p.seg_expert = pr.seg_expert;
  p.nseg = pr.nseg;
  p.num_mats = pr.num_mats;
  p.q = static_cast<const uint8_t*>(pr.w.qweight);
  p.s = static_cast<const uint16_t*>(pr.w.scales);
  p.z = static_cast<const uint8_t*>(pr.w.zeros);
  p.err = pr.err;
  // most row blocks there can be, however the rows fall into segments
  const int64_t hit = std::min<int64_t>(pr.nseg, pr.rows_cap);
  const int64_t u8 = hit + pr.rows_cap / 8, u16 = hit + pr.rows_cap / 16;
  switch (pr.w.group_size) {
    case 32: return launch_zeros<32>(p, pr.swiglu, u8, u16, st);
    case 64: return launch_zeros<64>(p, pr.swiglu, u8, u16, st);
    default: return launch_zeros<128>(p, pr.swiglu, u8, u16, st);
  }
}

}  // namespace prism
