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
// What bounds it: few rows reuse nothing, so every hit weight crosses HBM once and that is the floor.
// A block's warps split the inputs (kw ways) and keep their part of x in registers while the block
// streams its row tiles; the partial sums meet in shared memory in a fixed order. Blocks walk a
// device-side list of (segment, output tile, 8 * NT rows), so the host needs no counts.
#include <algorithm>

#include "internal.h"
#include "segments.cuh"
#include "w4.cuh"

namespace prism {
namespace {

constexpr int kWarps = 8;
constexpr int kSmallRows = 16;
constexpr int kCh = 2;          // 128-input chunks a warp keeps in registers per pass
constexpr int kColStride = 20;  // floats between the columns of a partial tile: no bank conflicts

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
  int blocks_n;              // ceil(tiles / rt)
  int64_t max_rows;          // longer segments are the other kernel's
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

template <int G, bool kZeros, bool kSwiGLU, int NT>
__global__ void __launch_bounds__(32 * kWarps, 2) w4_small_kernel(const SmallParams p) {
  constexpr int PG = 128 / G;   // groups per chunk
  extern __shared__ float smem[];
  int32_t* prefix = reinterpret_cast<int32_t*>(smem);
  float* part = smem + (p.nseg + 1 + 3) / 4 * 4;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int wk = warp % p.kw, wr = warp / p.kw;
  const int nwarps = blockDim.x >> 5;
  const int tile_floats = 8 * NT * kColStride;

  if (warp == 0) build_row_blocks(p.seg_offsets, p.nseg, p.rows_cap, 8 * NT, prefix, 0, p.max_rows);
  __syncthreads();
  const int64_t total = static_cast<int64_t>(prefix[p.nseg]) * p.blocks_n;

  for (int64_t item = blockIdx.x; item < total; item += gridDim.x) {
    const int sg = find_segment(prefix, p.nseg, static_cast<int32_t>(item / p.blocks_n));
    const int units = prefix[sg + 1] - prefix[sg];
    const int64_t rem = item - static_cast<int64_t>(prefix[sg]) * p.blocks_n;
    const int nb = static_cast<int>(rem / units), tb = static_cast<int>(rem % units);
    const RowSpan span = segment_rows(p.seg_offsets, sg, p.rows_cap);
    const int64_t row0 = span.begin + static_cast<int64_t>(tb) * 8 * NT;
    const int rows = static_cast<int>(min(static_cast<int64_t>(8 * NT), span.end - row0));
    const int e = p.seg_expert ? p.seg_expert[sg] : (p.num_mats == 1 ? 0 : sg);
    if (e < 0 || e >= p.num_mats) {   // an id no weights belong to: recorded, never read
      if (threadIdx.x == 0) record_device_error(p.err, PRISM_MOE_ERR_ARG);
      continue;
    }
    const int64_t mat = static_cast<int64_t>(e) * p.tiles;
    const int tile_end = min(p.tiles - nb * p.rt, p.rt);

    for (int pass = 0; pass < p.passes; ++pass) {
      const int c0 = (pass * p.kw + wk) * kCh;
      uint4 wq[2][kCh][2];
      auto load_tile = [&](int i, uint4(&w)[kCh][2]) {
        const int64_t base = (mat + nb * p.rt + i) * p.chunks;
#pragma unroll
        for (int c = 0; c < kCh; ++c)
          if (c0 + c < p.chunks) {
            const uint8_t* at = p.q + (base + c0 + c) * 1024 + lane * 16;
            w[c][0] = load_stream(at);
            w[c][1] = load_stream(at + 512);
          }
      };
      if (wr < tile_end) load_tile(wr, wq[0]);
      // this warp's part of x: rows g (+ 8 nt), inputs 8 t .. 8 t + 7 of each 32
      uint4 xb[kCh][NT][4];
#pragma unroll
      for (int c = 0; c < kCh; ++c)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int k = (c0 + c) * 128 + j * 32 + t * 8;
            const bool ok = g + 8 * nt < rows && k < p.K;
            xb[c][nt][j] = ok ? *reinterpret_cast<const uint4*>(p.x + (row0 + g + 8 * nt) * p.ld_x + k)
                              : make_uint4(0, 0, 0, 0);
          }
      int buf = 0;
#pragma unroll 1
      for (int i = wr; i < tile_end; i += p.rw, buf ^= 1) {
        uint4 w[kCh][2];
#pragma unroll
        for (int c = 0; c < kCh; ++c) {
          w[c][0] = wq[0][c][0];
          w[c][1] = wq[0][c][1];
        }
        if (i + p.rw < tile_end) load_tile(i + p.rw, wq[0]);
        float acc[NT][4] = {};
#pragma unroll
        for (int c = 0; c < kCh; ++c) {
          if (c0 + c >= p.chunks) continue;
          const int64_t chunk = (mat + nb * p.rt + i) * p.chunks + c0 + c;
          float sc[2][PG];
          uint32_t zr[2][PG];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int64_t at = (chunk * 16 + g + 8 * h) * PG;
            load_scales<PG>(p.s + at, sc[h]);
            load_zeros<PG, kZeros>(p.z, at, zr[h]);
          }
#pragma unroll
          for (int gr = 0; gr < PG; ++gr) {
            float part_acc[NT][4] = {};
#pragma unroll
            for (int j = gr * (4 / PG); j < (gr + 1) * (4 / PG); ++j) {
              const uint32_t w0 = word_of(w[c][0], j), w1 = word_of(w[c][1], j);
              uint32_t a[2][4];
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                a[0][q] = code_pair(w0, q, zr[0][gr]);
                a[1][q] = code_pair(w1, q, zr[1][gr]);
              }
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma_16816(part_acc[nt], a[0][0], a[1][0], a[0][1], a[1][1], xb[c][nt][j].x,
                          xb[c][nt][j].y);
                mma_16816(part_acc[nt], a[0][2], a[1][2], a[0][3], a[1][3], xb[c][nt][j].z,
                          xb[c][nt][j].w);
              }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              acc[nt][0] = fmaf(sc[0][gr], part_acc[nt][0], acc[nt][0]);
              acc[nt][1] = fmaf(sc[0][gr], part_acc[nt][1], acc[nt][1]);
              acc[nt][2] = fmaf(sc[1][gr], part_acc[nt][2], acc[nt][2]);
              acc[nt][3] = fmaf(sc[1][gr], part_acc[nt][3], acc[nt][3]);
            }
          }
        }
        float* mine = part + (wk * p.rt + i) * tile_floats;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float* at = mine + (8 * nt + 2 * t + (q & 1)) * kColStride + g + 8 * (q >> 1);
            *at = pass == 0 ? acc[nt][q] : *at + acc[nt][q];   // the same lane's own sum
          }
      }
    }
    __syncthreads();
    // sum of the kw partial tiles, two outputs per thread, neighbours along the output row
    constexpr int kPairs = kSwiGLU ? 4 : 8;   // output pairs of one row tile
    const int per_row = tile_end * kPairs;
    for (int i = threadIdx.x; i < rows * per_row; i += nwarps * 32) {
      const int col = i / per_row, pr = i % per_row;
      const int tile = pr / kPairs, r = pr % kPairs * 2;
      const float* at = part + tile * tile_floats + col * kColStride + r;
      float2 a = make_float2(0.f, 0.f), b = make_float2(0.f, 0.f);
      for (int k = 0; k < p.kw; ++k, at += p.rt * tile_floats) {
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
    __syncthreads();
  }
}

template <int G, bool kZeros, bool kSwiGLU, int NT>
int launch_small(SmallParams p, int64_t units, cudaStream_t st) {
  auto kern = w4_small_kernel<G, kZeros, kSwiGLU, NT>;
  // inputs: up to 8 warps x 2 chunks per pass; warps that the inputs do not need take row tiles
  p.passes = static_cast<int>(ceil_div(p.chunks, kWarps * kCh));
  p.kw = static_cast<int>(ceil_div(p.chunks, p.passes * kCh));
  p.rw = std::max(1, kWarps / p.kw);
  const int sms = num_sms();
  // row tiles per item: long items reuse x and amortise the joining of partial sums, short ones
  // fill the GPU when the call is small
  p.rt = p.rw;
  while (p.rt * 2 <= 8 && units * ceil_div(p.tiles, p.rt * 2) >= 4 * sms) p.rt *= 2;
  p.blocks_n = static_cast<int>(ceil_div(p.tiles, p.rt));
  const int bytes = static_cast<int>(sizeof(float)) *
                    ((p.nseg + 4) / 4 * 4 + p.kw * p.rt * 8 * NT * kColStride);
  constexpr int kMaxBytes = 4 * ((kMaxW4Segments + 4) + 8 * 8 * 8 * NT * kColStride);
  if (int r = ensure_smem_attr(reinterpret_cast<const void*>(kern), kMaxBytes)) return r;
  const int64_t items = units * p.blocks_n;
  const int grid = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(items, 2 * sms)));
  kern<<<grid, 32 * p.kw * p.rw, bytes, st>>>(p);
  PRISM_LAUNCH_CHECK("w4_small_kernel launch");
  return PRISM_MOE_OK;
}

template <int G, bool kZeros, bool kSwiGLU>
int launch_rows(const SmallParams& p, int64_t units8, int64_t units16, cudaStream_t st) {
  // 16 rows at a time once segments average more than 8
  if (p.rows_cap > 8 * static_cast<int64_t>(p.nseg))
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
  // Segments of at most kSmallRows rows run here, longer ones on the other kernel; the host does
  // not know the segments' lengths, so a call whose rows could make both kinds launches both.
  if (pr.rows_cap > kSmallRows)
    if (int r = w4_product_large(pr, kSmallRows, st)) return r;
  if (pr.nseg == 1 && pr.rows_cap > kSmallRows && !pr.seg_offsets) return PRISM_MOE_OK;
  SmallParams p{};
  p.max_rows = kSmallRows;
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
  const int64_t u8 = std::min(hit + pr.rows_cap / 8, 2 * hit), u16 = hit;
  switch (pr.w.group_size) {
    case 32: return launch_zeros<32>(p, pr.swiglu, u8, u16, st);
    case 64: return launch_zeros<64>(p, pr.swiglu, u8, u16, st);
    default: return launch_zeros<128>(p, pr.swiglu, u8, u16, st);
  }
}

}  // namespace prism
