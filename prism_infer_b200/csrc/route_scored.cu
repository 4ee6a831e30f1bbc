// Scored routing: softmax or sigmoid scores, a selection bias, expert groups, top-k, weights.
//
//   s_e   = softmax(l)_e  or  1 / (1 + exp(-l_e))
//   key_e = s_e + bias_e                       (the bias moves the choice, never the weight)
//   a group's score is its largest key, or the sum of its two largest; the topk_groups best stay
//   ids   = the k largest keys of the groups that stay, equal keys by ascending index
//   w_j   = s[ids_j] / (sum_j s[ids_j] + 1e-20) * scale   (the division only with renorm)
//
// One warp per token, keys in registers. A group's experts are spread over its own L lanes
// (L = 32 / next_pow2(groups)): lane g * L + j holds experts g * per + j + L * i, so a group's best
// keys meet in log2(L) shuffles whatever the sizes, and one group is the plain 32-lane layout.
// Keys are compared as order-preserving 64-bit integers (NaN above everything, as torch ranks it;
// 0 = no candidate): three warp-wide integer reductions find the best key and its lowest index.
#include "common.cuh"
#include "internal.h"

namespace prism {
namespace {

constexpr int kScoredWarps = 4;
constexpr unsigned kFull = 0xffffffffu;

template <bool kBf16>
__device__ __forceinline__ float load_logit(const void* p, int64_t i) {
  if constexpr (kBf16)
    return bf16_bits_to_float(reinterpret_cast<const uint16_t*>(p)[i]);
  else
    return reinterpret_cast<const float*>(p)[i];
}

__device__ __forceinline__ uint64_t order_key(double v) {
  if (isnan(v)) return ~0ull;
  const uint64_t b = static_cast<uint64_t>(__double_as_longlong(v + 0.0));   // -0 -> +0
  return (b >> 63) ? ~b : (b | (1ull << 63));
}
__device__ __forceinline__ double key_value(uint64_t k) {
  if (k == ~0ull) return __longlong_as_double(0x7ff8000000000000ll);
  return __longlong_as_double(static_cast<long long>((k >> 63) ? (k & ~(1ull << 63)) : ~k));
}

// Lowest ``idx`` among the lanes that hold the warp's largest ``key``.
__device__ __forceinline__ uint32_t warp_best(uint64_t key, uint32_t idx) {
  const uint32_t hi = static_cast<uint32_t>(key >> 32), lo = static_cast<uint32_t>(key);
  const uint32_t mh = __reduce_max_sync(kFull, hi);
  const uint32_t ml = __reduce_max_sync(kFull, hi == mh ? lo : 0u);
  return __reduce_min_sync(kFull, hi == mh && lo == ml ? idx : 0xffffffffu);
}

struct ScoredParams {
  const void* logits;
  const float* bias;
  int64_t T;
  int E, k, groups, keep, per, lanes;   // per = E / groups; lanes per group
  int sigmoid, top2, renorm;
  float scale;
  int64_t* ids;
  void* w;
  int w_bf16;
  int32_t* counts;
};

template <bool kBf16, int EPT>
__global__ void __launch_bounds__(32 * kScoredWarps) route_scored_kernel(const ScoredParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kScoredWarps + (threadIdx.x >> 5);
  if (t >= p.T) return;
  const int grp = lane / p.lanes, sub = lane % p.lanes;
  auto expert = [&](int i) { return grp * p.per + sub + p.lanes * i; };
  auto valid = [&](int i) { return grp < p.groups && sub + p.lanes * i < p.per; };

  float l[EPT];
  uint64_t key[EPT];
#pragma unroll
  for (int i = 0; i < EPT; ++i)
    l[i] = valid(i) ? load_logit<kBf16>(p.logits, t * p.E + expert(i)) : 0.f;

  // scores in 64 bits: the choice compares values that can lie closer than 32 bits resolve
  double top = 0.0, inv = 1.0;
  if (!p.sigmoid) {
    float m = -__int_as_float(0x7f800000);
#pragma unroll
    for (int i = 0; i < EPT; ++i)
      if (valid(i)) m = (l[i] > m || isnan(l[i])) ? l[i] : m;
    for (int off = 16; off > 0; off >>= 1) {
      const float o = __shfl_xor_sync(kFull, m, off);
      m = (o > m || isnan(o)) ? o : m;
    }
    top = m;
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < EPT; ++i)
      if (valid(i)) sum += exp(static_cast<double>(l[i]) - top);
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(kFull, sum, off);
    inv = sum;
  }
  auto score = [&](float v) {
    return p.sigmoid ? 1.0 / (1.0 + exp(-static_cast<double>(v)))
                     : exp(static_cast<double>(v) - top) / inv;
  };
#pragma unroll
  for (int i = 0; i < EPT; ++i) {
    key[i] = 0;
    if (valid(i))
      key[i] = order_key(score(l[i]) + (p.bias ? static_cast<double>(p.bias[expert(i)]) : 0.0));
  }

  // ---- groups: the keep best, equal scores by ascending group
  if (p.groups > 1) {
    uint64_t a = 0, b = 0;
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      const uint64_t lo = key[i] < a ? key[i] : a;
      a = key[i] > a ? key[i] : a;
      b = lo > b ? lo : b;
    }
    for (int off = p.lanes >> 1; off > 0; off >>= 1) {
      const uint64_t oa = __shfl_xor_sync(kFull, a, off), ob = __shfl_xor_sync(kFull, b, off);
      const uint64_t lo = oa < a ? oa : a, hb = ob > b ? ob : b;
      a = oa > a ? oa : a;
      b = lo > hb ? lo : hb;
    }
    uint64_t gs = 0;
    if (grp < p.groups) gs = p.top2 && p.per > 1 ? order_key(key_value(a) + key_value(b)) : a;
    int rank = 0;
    for (int g = 0; g < p.groups; ++g) {
      const uint64_t o = __shfl_sync(kFull, gs, g * p.lanes);
      rank += (o > gs || (o == gs && g < grp)) ? 1 : 0;
    }
    if (rank >= p.keep) {
#pragma unroll
      for (int i = 0; i < EPT; ++i) key[i] = 0;
    }
  }

  // ---- the k largest keys
  int my_i = 0;
  double my_s = 0.0;
  for (int j = 0; j < p.k; ++j) {
    uint64_t best = 0;
    int at = 0;
#pragma unroll
    for (int i = 0; i < EPT; ++i)
      if (key[i] > best) {   // a lane's experts ascend with i: the lowest index wins
        best = key[i];
        at = i;
      }
    const uint32_t mine = static_cast<uint32_t>(expert(at));
    const uint32_t win = warp_best(best, best ? mine : 0xfffffffeu);
    const bool owner = best != 0 && mine == win;
    float lv = 0.f;
#pragma unroll
    for (int i = 0; i < EPT; ++i)
      if (i == at) {
        lv = l[i];
        if (owner) key[i] = 0;
      }
    lv = __shfl_sync(kFull, lv, __ffs(__ballot_sync(kFull, owner)) - 1);
    if (lane == j) {
      my_i = static_cast<int>(win);
      my_s = score(lv);
    }
  }

  if (p.renorm) {
    double sum = lane < p.k ? my_s : 0.0;
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(kFull, sum, off);
    my_s /= sum + 1e-20;
  }
  if (lane < p.k) {
    const float w = static_cast<float>(my_s * static_cast<double>(p.scale));
    p.ids[t * p.k + lane] = my_i;
    if (p.w_bf16)
      reinterpret_cast<uint16_t*>(p.w)[t * p.k + lane] = float_to_bf16_bits(w);
    else
      reinterpret_cast<float*>(p.w)[t * p.k + lane] = w;
    if (p.counts) atomicAdd(p.counts + my_i, 1);
  }
}

template <bool kBf16>
int launch_scored(const ScoredParams& p, int ept, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>(ceil_div(p.T, kScoredWarps)));
  const dim3 block(32 * kScoredWarps);
#define PRISM_SCORED_CASE(N)                                   \
  if (ept <= N) {                                              \
    route_scored_kernel<kBf16, N><<<grid, block, 0, st>>>(p);  \
    PRISM_LAUNCH_CHECK("route_scored_kernel launch");          \
    return PRISM_MOE_OK;                                       \
  }
  PRISM_SCORED_CASE(1)
  PRISM_SCORED_CASE(2)
  PRISM_SCORED_CASE(4)
  PRISM_SCORED_CASE(8)
  PRISM_SCORED_CASE(16)
  PRISM_SCORED_CASE(32)
  PRISM_SCORED_CASE(64)
#undef PRISM_SCORED_CASE
  set_error("route_scored: %d experts in %d groups unsupported", p.E, p.groups);
  return PRISM_MOE_ERR_UNSUPPORTED;
}

}  // namespace

int route_scored(const void* logits, int dtype, int64_t T, int E, int k,
                 const prism_moe_router& r, int64_t* ids, void* w, int w_dtype, int32_t* counts,
                 cudaStream_t st) {
  if (counts) PRISM_CUDA(cudaMemsetAsync(counts, 0, sizeof(int32_t) * E, st));
  if (T == 0) return PRISM_MOE_OK;
  ScoredParams p{};
  p.logits = logits;
  p.bias = r.bias;
  p.T = T;
  p.E = E;
  p.k = k;
  p.groups = r.num_groups;
  p.keep = r.topk_groups;
  p.per = E / r.num_groups;
  int p2 = 1;
  while (p2 < r.num_groups) p2 <<= 1;
  p.lanes = 32 / p2;
  p.sigmoid = r.scoring == PRISM_MOE_SCORE_SIGMOID;
  p.top2 = r.group_score == PRISM_MOE_GROUP_TOP2;
  p.renorm = r.renorm;
  p.scale = r.scale;
  p.ids = ids;
  p.w = w;
  p.w_bf16 = w_dtype == PRISM_MOE_BF16;
  p.counts = counts;
  const int ept = static_cast<int>(ceil_div(p.per, p.lanes));
  return dtype == PRISM_MOE_BF16 ? launch_scored<true>(p, ept, st)
                                 : launch_scored<false>(p, ept, st);
}

}  // namespace prism
