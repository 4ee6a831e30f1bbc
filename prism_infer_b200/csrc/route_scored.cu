// Scored routing: softmax or sigmoid scores, a selection bias, expert groups, top-k, weights.
//
//   s_e   = softmax(l)_e  or  1 / (1 + exp(-l_e))
//   key_e = s_e + bias_e                       (the bias moves the choice, never the weight)
//   a group's score is its largest key, or the sum of its two largest; the topk_groups best stay
//   ids   = the k largest keys of the groups that stay, equal keys by ascending index
//   w_j   = s[ids_j] / (sum_j s[ids_j] + 1e-20) * scale   (the division only with renorm)
//
// One warp per token, keys in registers. A group's experts are spread over its own L lanes
// (L = 32 / next_pow2(groups)), consecutive ones on each, so a group's best keys meet in log2(L)
// shuffles whatever the sizes, and a lane reads its logits in vectors.
// Keys are compared as order-preserving integers (NaN above everything, as torch ranks it; 0 = no
// candidate); warp-wide integer reductions find the best key and its lowest index. Lanes of up to 8
// experts sort theirs first, so that taking the winner is a shift.
//
// The choice is that of 64-bit keys, made in 32 bits where those decide it. Without a bias the keys
// are the logits themselves (both scores increase with the logit), exactly; with one they are
// fp32 scores + bias, whose error is bounded. Any two neighbours in the order of the k + 1 best (and
// any two groups at the cut) that are closer than their errors, and not the same logit and bias,
// are looked at in 64 bits, and so is a tie at the cut with another key that close behind it: sigmoid
// keys with a bias among a few more candidates, all else (NaN,
// infinities and scores that saturate too) by choose_exact, on 64-bit keys of the whole row. On
// normal logits with a random bias about 1 row in 500 looks again, and nearly none goes on.
//
// What bounds it: 8192 tokens of 256 experts in 8 groups read 8.4 MB (1.4 us at the copy rate) and take
// 14.4 us on the GPU: the k + 1 rounds of two warp-wide reductions and the shuffles of the groups (SMs 53%
// busy, HBM 6%). One token takes 4 us more than an empty graph. 64-bit keys throughout took 29 us
// where these take 18 with a cold cache.
#include "common.cuh"
#include "internal.h"

namespace prism {
namespace {

constexpr int kScoredWarps = 4;
constexpr int kSpare = 4;   // candidates beyond the k that a close order looks at
constexpr unsigned kFull = 0xffffffffu;
constexpr float kFloor = 0x1p-120f;   // absolute error that any fp32 score is allowed, however small it is

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

__device__ __forceinline__ uint32_t order_key32(float v) {
  // adding zero makes -0 +0 and every NaN the canonical one, 0x7fffffff, whose key is ~0
  const uint32_t b = __float_as_uint(__fadd_rn(v, 0.f));
  return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value32(uint32_t k) {   // 0 (no candidate) reads as NaN
  return k == ~0u ? __int_as_float(0x7fc00000) : __uint_as_float((k >> 31) ? (k & 0x7fffffffu) : ~k);
}

// Two largest of a group's lanes.
template <typename Key>
__device__ __forceinline__ void join_top2(Key& a, Key& b, int lanes) {
  for (int off = lanes >> 1; off > 0; off >>= 1) {
    const Key oa = __shfl_xor_sync(kFull, a, off), ob = __shfl_xor_sync(kFull, b, off);
    const Key lo = oa < a ? oa : a, hb = ob > b ? ob : b;
    a = oa > a ? oa : a;
    b = lo > hb ? lo : hb;
  }
}

struct ScoredParams {
  const void* logits;
  const float* bias;
  int64_t T;
  int E, k, groups, keep, per, lanes, each;   // per = E / groups; lanes per group; experts per lane
  bool vec;   // a lane's logits and biases may be read in 16-byte vectors
  int sigmoid, top2, renorm;
  float scale;
  int64_t* ids;
  void* w;
  int w_bf16;
  int32_t* counts;
};

// A lane's ``mine`` consecutive values from element ``at`` on (0 beyond them).
template <bool kBf16, int EPT>
__device__ __forceinline__ void load_lane(const ScoredParams& p, const void* src, int64_t at,
                                          int mine, float (&v)[EPT]) {
  if constexpr (EPT >= 8 || (!kBf16 && EPT == 4)) {
    if (p.vec && mine == EPT) {
      if constexpr (kBf16) {
        const uint4* q = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(src) + at);
#pragma unroll
        for (int i = 0; i < EPT / 8; ++i) {
          const uint4 u = q[i];
          const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            v[8 * i + 2 * j] = __uint_as_float(w[j] << 16);
            v[8 * i + 2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
          }
        }
      } else {
        const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(src) + at);
#pragma unroll
        for (int i = 0; i < EPT / 4; ++i) {
          const float4 u = q[i];
          v[4 * i] = u.x;
          v[4 * i + 1] = u.y;
          v[4 * i + 2] = u.z;
          v[4 * i + 3] = u.w;
        }
      }
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < EPT; ++i) v[i] = i < mine ? load_logit<kBf16>(src, at + i) : 0.f;
}

struct Choice {
  int id;        // lane j: the j-th expert
  float logit;   // and its logit
};

// The choice from 64-bit keys (logits read again: rows come here rarely).
template <bool kBf16, int EPT>
__device__ __noinline__ Choice choose_exact(const ScoredParams& p, int64_t t) {
  const int lane = threadIdx.x & 31;
  const int grp = lane / p.lanes, sub = lane % p.lanes;
  auto expert = [&](int i) { return grp * p.per + sub * p.each + i; };
  auto valid = [&](int i) { return grp < p.groups && i < p.each && sub * p.each + i < p.per; };

  float l[EPT];
  uint64_t key[EPT];
#pragma unroll
  for (int i = 0; i < EPT; ++i)
    l[i] = valid(i) ? load_logit<kBf16>(p.logits, t * p.E + expert(i)) : 0.f;
  double top = 0.0, sum = 1.0;
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
    sum = 0.0;
#pragma unroll
    for (int i = 0; i < EPT; ++i)
      if (valid(i)) sum += exp(static_cast<double>(l[i]) - top);
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(kFull, sum, off);
  }
#pragma unroll
  for (int i = 0; i < EPT; ++i) {
    key[i] = 0;
    if (valid(i)) {
      const double s = p.sigmoid ? 1.0 / (1.0 + exp(-static_cast<double>(l[i])))
                                 : exp(static_cast<double>(l[i]) - top) / sum;
      key[i] = order_key(s + (p.bias ? static_cast<double>(p.bias[expert(i)]) : 0.0));
    }
  }
  if (p.keep < p.groups) {
    uint64_t a = 0, b = 0;
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      const uint64_t lo = key[i] < a ? key[i] : a;
      a = key[i] > a ? key[i] : a;
      b = lo > b ? lo : b;
    }
    join_top2(a, b, p.lanes);
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
  Choice mine{0, 0.f};
  for (int j = 0; j < p.k; ++j) {
    uint64_t best = 0;
    int at = 0;
#pragma unroll
    for (int i = 0; i < EPT; ++i)
      if (key[i] > best) {   // a lane's experts ascend with i: the lowest index wins
        best = key[i];
        at = i;
      }
    const uint32_t win = warp_best(best, best ? static_cast<uint32_t>(expert(at)) : 0xfffffffeu);
    const bool owner = best != 0 && static_cast<uint32_t>(expert(at)) == win;
    float lv = 0.f;
#pragma unroll
    for (int i = 0; i < EPT; ++i)
      if (i == at) {
        lv = l[i];
        if (owner) key[i] = 0;
      }
    lv = __shfl_sync(kFull, lv, __ffs(__ballot_sync(kFull, owner)) - 1);
    if (lane == j) mine = {static_cast<int>(win), lv};
  }
  return mine;
}

// Sort a lane's keys in descending order, equal keys by ascending index (odd-even transposition:
// N rounds of neighbours; N is 2, 4 or 8).
template <int N>
__device__ __forceinline__ void sort_lane(uint32_t (&key)[N], int (&at)[N]) {
#pragma unroll
  for (int r = 0; r < N; ++r)
#pragma unroll
    for (int i = r & 1; i + 1 < N; i += 2)
      if (key[i + 1] > key[i]) {   // neighbours never swap when equal: the order stays by index
        const uint32_t k = key[i];
        key[i] = key[i + 1];
        key[i + 1] = k;
        const int a = at[i];
        at[i] = at[i + 1];
        at[i + 1] = a;
      }
}

template <bool kBf16, int EPT>
__global__ void __launch_bounds__(32 * kScoredWarps) route_scored_kernel(const __grid_constant__ ScoredParams p) {
  constexpr bool kSorted = EPT <= 8;
  const int lane = threadIdx.x & 31;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kScoredWarps + (threadIdx.x >> 5);
  if (t >= p.T) return;
  const int grp = lane / p.lanes, sub = lane % p.lanes;
  const int first = grp * p.per + sub * p.each;
  const int mine = grp < p.groups ? max(0, min(p.each, p.per - sub * p.each)) : 0;   // this lane's experts

  float l[EPT];
  load_lane<kBf16, EPT>(p, p.logits, t * p.E + first, mine, l);
  uint32_t key[EPT];
  int at[EPT];
  uint32_t top_key = 0;
#pragma unroll
  for (int i = 0; i < EPT; ++i) {
    at[i] = i;
    key[i] = i < mine ? order_key32(l[i]) : 0u;
    top_key = max(top_key, key[i]);
  }
  const float top = key_value32(__reduce_max_sync(kFull, top_key));   // largest logit, or NaN
  bool unsure = !(fabsf(top) <= 3.4028235e38f);

  // ---- fp32 scores where they are needed: as keys with a bias, or for the sum of a softmax
  const bool need_sum = !p.sigmoid && (p.bias || !p.renorm);
  float sum = 1.f;
  if (need_sum) {
    float e[EPT];
#pragma unroll
    for (int i = 0; i < EPT; ++i) e[i] = i < mine ? expf(l[i] - top) : 0.f;
#pragma unroll
    for (int w = EPT / 2; w > 0; w >>= 1)
#pragma unroll
      for (int i = 0; i < w; ++i) e[i] += e[i + w];
    sum = e[0];
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(kFull, sum, off);
  }
  auto score = [&](float v) {
    return p.sigmoid ? __fdividef(1.f, 1.f + expf(-v)) : __fdividef(expf(v - top), sum);
  };
  if (p.bias) {
    float b[EPT];
    load_lane<false, EPT>(p, p.bias, first, mine, b);
#pragma unroll
    for (int i = 0; i < EPT; ++i)
      if (i < mine) key[i] = order_key32(score(l[i]) + b[i]);
  }
  // Error of any fp32 score of this row. Sigmoid: expf (2 ulp), a sum and a division (2 ulp), 2^-20
  // of the score. Softmax: expf, its argument (|l - top| 2^-24, but e^-x x < 0.4), a division and a sum
  // whose 2^6 lane terms and 32 lanes meet in a tree (11 roundings): 2^-19 of the largest.
  // Scores under 2^-126 come out as 0 (expf(-l) above 2^126 makes the division 0): kFloor covers them.
  const float score_err = p.bias ? fmaf(p.sigmoid ? 0x1p-20f : 0x1p-19f, score(top), kFloor) : 0.f;
  if constexpr (kSorted && EPT > 1) sort_lane(key, at);

  // ---- groups: the keep best, equal scores by ascending group
  if (p.keep < p.groups) {   // else there is no cut, and nothing to be unsure of
    uint32_t a = 0, b = 0;
    if constexpr (kSorted) {
      a = key[0];
      if constexpr (EPT > 1) b = key[1];
    } else {
#pragma unroll
      for (int i = 0; i < EPT; ++i) {
        const uint32_t lo = min(key[i], a);
        a = max(a, key[i]);
        b = max(b, lo);
      }
    }
    join_top2(a, b, p.lanes);
    const bool two = p.top2 && p.per > 1;
    const float va = key_value32(a), vb = two ? key_value32(b) : 0.f;
    float gs = va, err = 0.f;
    if (p.bias) {
      gs = va + vb;
      err = 2.f * score_err + 0x1p-22f * (fabsf(va) + fabsf(vb));
    } else if (two) {   // keys are logits: their scores, up to the softmax's common factor
      gs = p.sigmoid ? score(va) + score(vb) : expf(va - top) + expf(vb - top);
      err = p.sigmoid ? fmaf(0x1p-20f, gs, kFloor) : 0x1p-20f;
    }
    int rank = 0;
    for (int g = 0; g < p.groups; ++g) {
      const float o = __shfl_sync(kFull, gs, g * p.lanes);
      rank += (o > gs || (o == gs && g < grp)) ? 1 : 0;
    }
    const bool kept = grp < p.groups && rank < p.keep;
    // certain where the worst that stays and the best that goes are further apart than their errors
    float low = kept ? gs - err : __int_as_float(0x7f800000);
    float high = grp < p.groups && !kept ? gs + err : -__int_as_float(0x7f800000);
    for (int off = 16; off > 0; off >>= 1) {
      low = fminf(low, __shfl_xor_sync(kFull, low, off));
      high = fmaxf(high, __shfl_xor_sync(kFull, high, off));
    }
    const bool exact = !p.bias && !two;   // logits: equal ones are ties, distinct ones decided
    // (lanes of no group hold no score)
    unsure |= !(low > high || (exact && low == high)) || (grp < p.groups && !(gs == gs));
    if (exact)
      // (a tie at the cut: no other group may be that close to it)
      unsure |= (low - high > 0.f && low - high < 0x1p-40f) ||
                (low == high && grp < p.groups && gs != low && fabsf(gs - low) < 0x1p-40f) ||
                (p.sigmoid ? fabsf(low) > 16.f : !(top - low <= 600.f));   // saturated
    if (!kept) {
#pragma unroll
      for (int i = 0; i < EPT; ++i) key[i] = 0;
    }
  }

  // ---- the k largest keys, and the next one to compare with
  uint32_t next_key = 0, next_id = 0;
  auto take_next = [&]() {   // the warp's best key and its lowest index, taken off its lane
    uint32_t best = 0;
    int pos = 0;
    if constexpr (kSorted) {
      best = key[0];
      pos = at[0];
    } else {
#pragma unroll
      for (int i = 0; i < EPT; ++i)
        if (key[i] > best) {
          best = key[i];
          pos = i;
        }
    }
    next_key = __reduce_max_sync(kFull, best);
    const uint32_t id = static_cast<uint32_t>(first + pos);
    next_id = __reduce_min_sync(kFull, best == next_key ? id : 0xffffffffu);
    if (best == next_key && id == next_id) {
      if constexpr (kSorted) {
#pragma unroll
        for (int i = 0; i + 1 < EPT; ++i) {
          key[i] = key[i + 1];
          at[i] = at[i + 1];
        }
        key[EPT - 1] = 0;
      } else {
#pragma unroll
        for (int i = 0; i < EPT; ++i)
          if (i == pos) key[i] = 0;
      }
    }
  };
  uint32_t my_key = 0;
  Choice my{0, 0.f};
  for (int j = 0; j <= p.k; ++j) {
    take_next();
    if (lane == j) {
      my_key = next_key;
      my.id = static_cast<int>(next_id);
    }
  }
  if (lane >= p.k) {   // every other lane stands for the next one (key 0: there is none)
    my_key = next_key;
    my.id = static_cast<int>(next_id);
  }
  const bool have = my_key != 0;
  if (have) my.logit = load_logit<kBf16>(p.logits, t * p.E + my.id);   // in the cache
  const float v = key_value32(my_key), mb = have && p.bias ? p.bias[my.id] : 0.f;
  float nv = __shfl_down_sync(kFull, v, 1), nl = __shfl_down_sync(kFull, my.logit, 1);
  float nb = __shfl_down_sync(kFull, mb, 1);
  if (p.k == 32 && lane == 31) {
    nv = key_value32(next_key);
    nl = next_key ? load_logit<kBf16>(p.logits, t * p.E + next_id) : 0.f;
    nb = next_key && p.bias ? p.bias[next_id] : 0.f;
  }
  auto reach = [&](float x, float y) {   // two keys closer than this may be in the wrong order
    return 2.f * score_err + 0x1p-22f * (fabsf(x) + fabsf(y));
  };
  bool close = false;   // in the wrong order, perhaps
  bool tie = false;     // equal in 64 bits too, and others may be close
  if (lane < p.k) {
    const bool next = lane + 1 < p.k || next_key != 0;
    if (p.bias) {
      tie = next && my.logit == nl && mb == nb;
      if (next) close = !(v - nv > reach(v, nv)) && !tie;
      unsure |= !(fabsf(v) <= 3.4028235e38f);
    } else {
      // where 64-bit scores could merge distinct logits: next to 0 or 1, or next to each other
      tie = next && v == nv && fabsf(v) < 0x1p-16f;   // larger ones lie 2^-40 apart or more
      if (next) unsure |= v - nv > 0.f && v - nv < 0x1p-40f;
      unsure |= p.sigmoid ? !(fabsf(v) <= 16.f) : !(top - v <= 600.f);
    }
  }
  if (__shfl_sync(kFull, tie, p.k - 1)) {
    // A tie at the cut says nothing of the keys behind it: one of another logit or bias that is in
    // reach of the tied ones may belong before them.
    const float cut = __shfl_sync(kFull, v, p.k - 1), cut_logit = __shfl_sync(kFull, my.logit, p.k - 1);
    const float cut_bias = __shfl_sync(kFull, mb, p.k - 1);
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      const float o = key_value32(key[i]);
      if (key[i] == 0 || o == -__int_as_float(0x7f800000)) continue;   // far from a finite cut
      if (!p.bias) {
        unsure |= o < cut && cut - o < 0x1p-40f;
      } else if (!(cut - o > reach(cut, o))) {
        const int id = first + at[i];
        close |= !(load_logit<kBf16>(p.logits, t * p.E + id) == cut_logit && p.bias[id] == cut_bias);
      }
    }
  }
  unsure = __any_sync(kFull, unsure);
  if (__any_sync(kFull, close) && !unsure) {
    // Sigmoid keys need no other expert's: a few more candidates, all of them in 64 bits, one to a
    // lane, and the order is certain where the last one is out of reach of the k-th.
    const int m = p.k + kSpare;
    unsure = !p.sigmoid || m > 32;
    if (!unsure) {
      for (int j = p.k + 1; j < m; ++j) {
        take_next();
        if (lane == j) {
          my_key = next_key;
          my.id = static_cast<int>(next_id);
        }
      }
      const bool there = lane < m && my_key != 0;
      double key64 = 0.0;
      if (there) {
        my.logit = load_logit<kBf16>(p.logits, t * p.E + my.id);
        key64 = 1.0 / (1.0 + exp(-static_cast<double>(my.logit))) + static_cast<double>(p.bias[my.id]);
      }
      const int n = __popc(__ballot_sync(kFull, there));
      int rank = lane;
      if (there) rank = 0;
      for (int i = 0; i < n; ++i) {
        const double o = __shfl_sync(kFull, key64, i);
        const int oid = __shfl_sync(kFull, my.id, i);
        if (there && (o > key64 || (o == key64 && oid < my.id))) ++rank;
      }
      int src = lane;
      for (int i = 0; i < n; ++i)
        if (__shfl_sync(kFull, rank, i) == lane) src = i;
      my.id = __shfl_sync(kFull, my.id, src);
      my.logit = __shfl_sync(kFull, my.logit, src);
      key64 = __shfl_sync(kFull, key64, src);
      if (n == m) {   // there may be more: none of them may reach the k-th
        const float last = key_value32(next_key);
        const float kth = static_cast<float>(__shfl_sync(kFull, key64, p.k - 1));
        unsure = !(kth - last > 2.f * score_err + 0x1p-21f * (fabsf(kth) + fabsf(last)));
      }
    }
  }
  if (unsure) my = choose_exact<kBf16, EPT>(p, t);

  // ---- weights: scores of the chosen, the softmax's argument with the rounding of v - top put back
  float s = 0.f;
  if (lane < p.k) {
    if (p.sigmoid) {
      // far down the sum is e^-l itself, which overflows before its inverse is 0
      s = my.logit < -80.f ? expf(my.logit) : 1.f / (1.f + expf(-my.logit));
    } else {
      const float d = my.logit - top, z = d - my.logit;
      const float lost = (my.logit - (d - z)) - (top + z);
      const float e = expf(d);
      s = (lost == lost ? fmaf(e, lost, e) : e) / sum;   // a logit of -inf: e is 0
      // a NaN or infinite logit leaves no weight of its token a number, as in softmax itself
      if (!(fabsf(top) <= 3.4028235e38f)) s = __int_as_float(0x7fc00000);
    }
  }
  if (p.renorm) {
    float total = s;
    for (int off = 16; off > 0; off >>= 1) total += __shfl_xor_sync(kFull, total, off);
    s /= total + 1e-20f;
  }
  if (lane < p.k) {
    const float w = s * p.scale;
    p.ids[t * p.k + lane] = my.id;
    if (p.w_bf16)
      reinterpret_cast<uint16_t*>(p.w)[t * p.k + lane] = float_to_bf16_bits(w);
    else
      reinterpret_cast<float*>(p.w)[t * p.k + lane] = w;
    if (p.counts) atomicAdd(p.counts + my.id, 1);
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
  p.each = static_cast<int>(ceil_div(p.per, p.lanes));
  // rows, groups and lanes all start at multiples of 16 bytes of logits (and of 4 biases)
  const int unit = dtype == PRISM_MOE_BF16 ? 8 : 4;
  p.vec = E % unit == 0 && p.per % unit == 0 && p.each % unit == 0 &&
          (reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(r.bias)) % 16 == 0;
  return dtype == PRISM_MOE_BF16 ? launch_scored<true>(p, p.each, st)
                                 : launch_scored<false>(p, p.each, st);
}

}  // namespace prism
