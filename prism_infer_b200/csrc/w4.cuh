// 4-bit weights: the layout both product kernels read, and its decoding.
//
// A matrix [N, K] is held in tiles of 16 rows by 128 inputs, row tiles outermost:
//   qweight [N/16][ceil(K/128)][16 rows][64 bytes]      scales, zeros [N/16][ceil(K/128)][16][128/G]
// A row's 64 bytes are 16 words of 8 codes; the word at 4 t + j (t, j < 4) holds inputs
// 32 j + 8 t .. + 7, nibbles from the low end: inputs 0 2 4 6 1 3 5 7 of the eight. So a 16-byte load
// of quarter t gives, in word j, the 8 consecutive inputs that belong to group (32 j) / G, and
// (word >> 4 i) & 0x000f000f is the pair of inputs (2 i, 2 i + 1) in the two halves of a register.
// gate_up matrices alternate 8 gate rows and 8 up rows, so a tile holds both factors of 8 outputs.
#pragma once
#include "common.cuh"
#include "segments.cuh"

namespace prism {

__device__ __forceinline__ uint32_t word_of(const uint4& v, int j) {
  return j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w;
}

// bf16 pair (code - zero) of inputs (2 i, 2 i + 1); ``zero`` holds 128 + zero twice. Both the value
// 128 + code (128 .. 143, 7 fraction bits suffice) and the difference are exact.
__device__ __forceinline__ uint32_t code_pair(uint32_t word, int i, uint32_t zero) {
  uint32_t c, d;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(c) : "r"(word >> (4 * i)), "r"(0x000f000fu), "r"(0x43004300u));
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(c), "r"(zero));
  return d;
}

// bf16 pair offset + code of inputs (2 i, 2 i + 1). Nibbles in bits 0-3 of a half, as they are or
// after a shift by 8, are the lowest of the seven fraction bits under the exponent of 128 (i = 0, 2);
// nibbles in bits 4-7 move down by one bit to the highest under the exponent of 16 (i = 1, 3). Mask
// and exponent go in with one three-input operation. Without kMixed every nibble goes under 16.
template <bool kMixed>
__device__ __forceinline__ uint32_t offset_pair(uint32_t word, int i) {
  const bool low = kMixed && !(i & 1);
  const uint32_t c = low ? (i ? word >> 8 : word) : i == 0 ? word << 3 : word >> (4 * i - 3);
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;"
      : "=r"(d)
      : "r"(c), "r"(low ? 0x000f000fu : 0x00780078u), "r"(low ? 0x43004300u : 0x41804180u));
  return d;
}

// The PG scales of one row and chunk (global or shared memory), widened to fp32 (exact).
template <int PG>
__device__ __forceinline__ void load_scales(const uint16_t* p, float (&s)[PG]) {
  if constexpr (PG == 1) {
    s[0] = bf16_bits_to_float(*p);
  } else if constexpr (PG == 2) {
    const uint32_t v = *reinterpret_cast<const uint32_t*>(p);
    s[0] = __uint_as_float(v << 16);
    s[1] = __uint_as_float(v & 0xffff0000u);
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    s[0] = __uint_as_float(v.x << 16);
    s[1] = __uint_as_float(v.x & 0xffff0000u);
    s[2] = __uint_as_float(v.y << 16);
    s[3] = __uint_as_float(v.y & 0xffff0000u);
  }
}

// The zero point of each of the PG groups.
template <int PG>
__device__ __forceinline__ void load_zero_points(const uint8_t* z, float (&out)[PG]) {
  uint32_t v;
  if constexpr (PG == 1)
    v = *z;
  else if constexpr (PG == 2)
    v = *reinterpret_cast<const uint16_t*>(z);
  else
    v = *reinterpret_cast<const uint32_t*>(z);
#pragma unroll
  for (int i = 0; i < PG; ++i) out[i] = static_cast<float>((v >> (8 * i)) & 0xfu);
}

// silu(g) * u in fp32, with the fast exponential and division: off by 2^-16 of the result at most for
// |g| <= 87 (below -87 it is 0, where the result is under 2^-119 of u), and rounded to bf16 next.
__device__ __forceinline__ float silu_mul(float g, float u) {
  return __fdividef(g, 1.f + __expf(-g)) * u;
}

// Programmatic launches: wait for the end (and the writes) of the kernel before this one; let the
// next one start once every block has come here or ended.
__device__ __forceinline__ void wait_for_earlier() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
__device__ __forceinline__ void launch_dependents() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

struct RowSpan {
  int64_t begin, end;
};

// Rows of segment s, kept inside [0, rows_cap) (no table: one segment of every row).
__device__ __forceinline__ RowSpan segment_rows(const int32_t* seg_offsets, int s,
                                                int64_t rows_cap) {
  if (!seg_offsets) return {0, rows_cap};
  const int64_t b = max(seg_offsets[s], 0);
  return {b, min(static_cast<int64_t>(seg_offsets[s + 1]), rows_cap)};
}

// Warp-cooperative: prefix[s] = row blocks (of ``bm`` rows) before segment s, prefix[nseg] = all.
// Only segments of more than ``min_rows`` rows count.
__device__ __forceinline__ void build_row_blocks(const int32_t* seg_offsets, int nseg,
                                                 int64_t rows_cap, int bm, int32_t* prefix,
                                                 int64_t min_rows) {
  const int lane = threadIdx.x & 31;
  int32_t carry = 0;
  for (int base = 0; base < nseg; base += 32) {
    const int s = base + lane;
    int32_t n = 0;
    if (s < nseg) {
      const RowSpan r = segment_rows(seg_offsets, s, rows_cap);
      const int64_t len = r.end - r.begin;
      n = len > min_rows ? static_cast<int32_t>((len + bm - 1) / bm) : 0;
    }
    int32_t incl = n;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int32_t y = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += y;
    }
    if (s < nseg) prefix[s] = carry + incl - n;
    carry += __shfl_sync(0xffffffffu, incl, 31);
  }
  if (lane == 0) prefix[nseg] = carry;
}

// The same by all threads of a block (at most 1024 segments, blocks of up to 256 threads), counting
// segments of at most ``max_rows`` rows: every offset is loaded at once, so the list costs one memory
// latency. Ends with a barrier.
__device__ __forceinline__ void build_row_blocks_cta(const int32_t* seg_offsets, int nseg,
                                                     int64_t rows_cap, int bm, int32_t* prefix,
                                                     int64_t max_rows) {
  __shared__ int32_t warp_sum[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int each = (nseg + blockDim.x - 1) / blockDim.x;
  const int first = threadIdx.x * each;
  int32_t mine = 0;
  for (int i = 0; i < each; ++i)
    if (first + i < nseg) {
      const RowSpan r = segment_rows(seg_offsets, first + i, rows_cap);
      const int64_t len = r.end - r.begin;
      const int32_t b = len > 0 && len <= max_rows ? static_cast<int32_t>((len + bm - 1) / bm) : 0;
      prefix[first + i] = mine;   // within this thread's run
      mine += b;
    }
  int32_t incl = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int32_t y = __shfl_up_sync(0xffffffffu, incl, off);
    if (lane >= off) incl += y;
  }
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  int32_t before = incl - mine;
  for (int w = 0; w < warp; ++w) before += warp_sum[w];
  for (int i = 0; i < each; ++i)
    if (first + i < nseg) prefix[first + i] += before;
  if (threadIdx.x == blockDim.x - 1) prefix[nseg] = before + mine;
  __syncthreads();
}

}  // namespace prism
