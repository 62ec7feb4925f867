// Expert choice from router logits, one warp per token (many rows of 16-bit
// logits alone: one thread, see there).
//
//   s = softmax(l) or 1 / (1 + exp(-l))            score of each expert
//   c = s + bias, and -inf where l = -inf          what the choice goes by
//   worth(group) = max c, or the sum of its two largest c (a missing second
//   one counts 0); experts outside the best `topk_group` groups get c = -inf
//   ids = the k largest c in descending order;  w = s[ids] (/ sum) * scale
// Equal values go by the larger logit, then by the lower index (equal groups by
// the logit of their best expert, then by index). A slot for which no expert is left
// (c = -inf) gets id E and weight 0: the expert forwards skip ids outside
// [0, E). A row with a NaN logit or choice (softmax: or a +inf logit) gets
// NaN weights for ids 0..k-1, so that the NaN reaches the layer's output.
//
// The ids are those of 64-bit arithmetic. Without a bias both scores rise
// with the logit, so the choice compares the logits themselves (softmax
// probabilities of one row, and sigmoids, order as their logits do; group
// maxima too). With a bias, or with top-2 group sums, the warp compares f32
// values and notes whether any comparison that decided was closer than
// their error bound; such a row (about one in a thousand at 256 experts and
// normal logits) is done again in 64 bits. There sigmoids of all logits from
// about 37 on are 1, and small scores vanish beside a bias: that equal values
// go by their logits makes a bias that is the same for all change nothing.
//
// Layout: lane L holds the experts L*PER .. L*PER+PER-1, so a row is read
// with wide loads and the lowest lane that holds a maximum also holds the
// lowest index. Per choice: the lane's maximum of PER keys, one redux.sync,
// one ballot.
#include <algorithm>

#include "common.cuh"

namespace aeoq {

constexpr int kRouteWarps = 4;        // rows per block
constexpr int kRouteMaxExperts = 1024;
constexpr int kRouteMaxK = 32;
constexpr int kRouteMaxGroups = 32;

struct RouteParams {
  const void* logits;
  int64_t ld, T;
  int E, k;
  const float* bias;     // null: none
  int n_group, topk_group;
  int sigmoid, top2, renorm;
  int vec;               // rows may be read in PER-wide pieces
  float scale;
  float* w;
  int64_t* ids;
};

// Floats as unsigned integers of the same order; -inf is 0x007FFFFF, so 0 is
// free for "no such expert, or already taken".
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t b = __float_as_uint(v);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float order_val(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}
constexpr uint32_t kNegInfKey = 0x007FFFFFu;

__device__ __forceinline__ uint64_t order_key64(double v) {
  const uint64_t b = (uint64_t)__double_as_longlong(v);
  return (b >> 63) ? ~b : (b | (1ull << 63));
}
__device__ __forceinline__ double order_val64(uint64_t k) {
  return __longlong_as_double((long long)((k >> 63) ? (k & 0x7FFFFFFFFFFFFFFFull) : ~k));
}
constexpr uint64_t kNegInfKey64 = 0x000FFFFFFFFFFFFFull;

__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}
__device__ __forceinline__ uint64_t warp_max64(uint64_t v) {
  const uint32_t hi = __reduce_max_sync(0xFFFFFFFFu, (uint32_t)(v >> 32));
  const uint32_t lo = __reduce_max_sync(0xFFFFFFFFu, (uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
  return ((uint64_t)hi << 32) | lo;
}

template <int DT>
__device__ __forceinline__ float route_logit(const RouteParams& p, int64_t row, int e) {
  return In<DT>::load(reinterpret_cast<const typename In<DT>::T*>(p.logits) + row * p.ld + e);
}

// A logit as an ordered key (-0 and +0 are equal).
template <int DT>
__device__ __forceinline__ uint32_t route_logit_key(const RouteParams& p, int64_t row, int e) {
  return order_key(route_logit<DT>(p, row, e) + 0.0f);
}

// Which groups stay: bit g of the result. Lane g holds group g's worth and, with
// BY_LOGIT, the key of its best expert's logit. `near` is set where a kept and a
// dropped group are within tol of one another (in 64 bits: equal).
template <class Val, bool BY_LOGIT = false>
__device__ __forceinline__ uint32_t keep_groups(Val worth, int n_group, int topk_group, Val tol, bool& near,
                                                uint32_t lead = 0) {
  const int lane = threadIdx.x & 31;
  int rank = 0;
  for (int h = 0; h < n_group; ++h) {
    const Val o = __shfl_sync(0xFFFFFFFFu, worth, h);
    if constexpr (BY_LOGIT) {
      const uint32_t l = __shfl_sync(0xFFFFFFFFu, lead, h);
      rank += o > worth || (o == worth && (l > lead || (l == lead && h < lane)));
    } else {
      rank += (o > worth) || (o == worth && h < lane);
    }
  }
  const uint32_t keep = __ballot_sync(0xFFFFFFFFu, lane < n_group && rank < topk_group);
  bool mine = false;
  for (int h = 0; h < n_group; ++h) {
    const Val o = __shfl_sync(0xFFFFFFFFu, worth, h);
    if constexpr (sizeof(Val) == 8) {
      mine |= lane < n_group && (((keep >> h) ^ (keep >> lane)) & 1u) && o == worth && worth > -INFINITY;
    } else {
      const Val d = o > worth ? o - worth : worth - o;       // inf - inf is NaN: not near
      mine |= lane < n_group && (((keep >> h) ^ (keep >> lane)) & 1u) && d <= tol;
    }
  }
  near = __any_sync(0xFFFFFFFFu, mine);
  return keep;
}

// One row in 64 bits: the same definition, plainly. Rows come here when f32
// cannot tell two choices apart, or when every chosen score is so small that
// f32 has lost it. Without BY_LOGIT it stops where two values are equal that
// the choice may be between, and returns true: the row is then done with it.
template <int PER, int DT, bool ONLY_LOGITS, bool BY_LOGIT>
__device__ __noinline__ bool route_row64(const RouteParams& p, int64_t row) {
  // (with it, small code: few rows come here twice)
  constexpr int kUnroll = BY_LOGIT ? 1 : PER;
  const int lane = threadIdx.x & 31;
  double s[PER];
  uint64_t key[PER];
  double m = -INFINITY;
#pragma unroll kUnroll
  for (int i = 0; i < PER; ++i) {
    const int e = lane * PER + i;
    s[i] = e < p.E ? (double)route_logit<DT>(p, row, e) : -INFINITY;
    m = fmax(m, s[i]);
  }
  double total = 1.0;
  if (!p.sigmoid) {
    m = order_val64(warp_max64(order_key64(m)));
    if (m == -INFINITY) m = 0.0;
    double t = 0.0;
#pragma unroll kUnroll
    for (int i = 0; i < PER; ++i) t += exp(s[i] - m);
    total = warp_sum64(t);
  }
#pragma unroll kUnroll
  for (int i = 0; i < PER; ++i) {
    const int e = lane * PER + i;
    const double l = s[i];
    s[i] = p.sigmoid ? 1.0 / (1.0 + exp(-l)) : (total > 0.0 ? exp(l - m) / total : 0.0);
    const double c = ONLY_LOGITS || l == -INFINITY ? l : s[i] + (p.bias && e < p.E ? (double)p.bias[e] : 0.0);
    key[i] = e < p.E ? order_key64(c + 0.0) : 0ull;
  }
  if (p.n_group > 1) {
    const int S = p.E / p.n_group;
    double worth = -INFINITY;
    const int lpg = S / PER;
    const bool whole = S % PER == 0 && (lpg & (lpg - 1)) == 0;
    if (whole) {
      uint64_t a = 0, b = 0;
#pragma unroll kUnroll
      for (int i = 0; i < PER; ++i) {
        if (key[i] > a) { b = a; a = key[i]; }
        else if (key[i] > b) b = key[i];
      }
      for (int o = 1; o < lpg; o <<= 1) {
        const uint64_t c = __shfl_xor_sync(0xFFFFFFFFu, a, o), d = __shfl_xor_sync(0xFFFFFFFFu, b, o);
        const uint64_t low = a < c ? a : c;
        b = b > d ? b : d;
        b = b > low ? b : low;
        a = a > c ? a : c;
      }
      double v = order_val64(a);
      if (p.top2 && b > kNegInfKey64) v += order_val64(b);
      worth = __shfl_sync(0xFFFFFFFFu, v, lane * lpg);
      if (lane >= p.n_group) worth = -INFINITY;
    }
    for (int g = 0; g < p.n_group && !whole; ++g) {
      uint64_t a = 0, b = 0;
#pragma unroll kUnroll
      for (int i = 0; i < PER; ++i) {
        const int e = lane * PER + i;
        if (e >= g * S && e < (g + 1) * S) {
          if (key[i] > a) { b = a; a = key[i]; }
          else if (key[i] > b) b = key[i];
        }
      }
      const uint64_t ga = warp_max64(a);
      const int who = __ffs(__ballot_sync(0xFFFFFFFFu, a == ga)) - 1;
      const uint64_t gb = warp_max64(lane == who ? b : a);
      double v = order_val64(ga);
      if (p.top2 && gb > kNegInfKey64) v += order_val64(gb);
      if (lane == g) worth = v;
    }
    bool near;
    uint32_t lead = 0;
    if constexpr (BY_LOGIT) {
      for (int g = 0; g < p.n_group; ++g) {
        uint64_t a = 0;
#pragma unroll kUnroll
        for (int i = 0; i < PER; ++i) {
          const int e = lane * PER + i;
          if (e >= g * S && e < (g + 1) * S && key[i] > a) a = key[i];
        }
        a = warp_max64(a);
        uint32_t equal = 0, l = 0;
#pragma unroll kUnroll
        for (int i = 0; i < PER; ++i) {
          const int e = lane * PER + i;
          equal |= (uint32_t)(e >= g * S && e < (g + 1) * S && key[i] == a) << i;
        }
        for (; equal; equal &= equal - 1) l = max(l, route_logit_key<DT>(p, row, lane * PER + __ffs(equal) - 1));
        l = __reduce_max_sync(0xFFFFFFFFu, l);
        if (lane == g) lead = l;
      }
    }
    const uint32_t keep = keep_groups<double, BY_LOGIT>(worth, p.n_group, p.topk_group, 0.0, near, lead);
    if (!BY_LOGIT && !ONLY_LOGITS && near) return true;
#pragma unroll kUnroll
    for (int i = 0; i < PER; ++i) {
      const int e = lane * PER + i;
      if (e < p.E && !((keep >> (e / S)) & 1u)) key[i] = kNegInfKey64;
    }
  }
  double my_w = 0.0;
  int my_id = p.E;
  uint64_t prev = 0;
  constexpr bool kLook = !BY_LOGIT && !ONLY_LOGITS;
  for (int j = 0; j < p.k + (int)kLook; ++j) {
    uint64_t best = 0;
#pragma unroll kUnroll
    for (int i = 0; i < PER; ++i) best = key[i] > best ? key[i] : best;
    const uint64_t top = warp_max64(best);
    if (top <= kNegInfKey64) break;
    if constexpr (kLook) {
      if (top == prev) return true;
      if (j == p.k) break;
      prev = top;
    }
    int at = 0;
    double sv = 0.0;
    int src;
    if constexpr (BY_LOGIT) {
      uint32_t equal = 0, mine = 0;      // which of this lane's have that value, their largest logit
#pragma unroll kUnroll
      for (int i = 0; i < PER; ++i) equal |= (uint32_t)(key[i] == top) << i;
      int pick = -1;
      for (; equal; equal &= equal - 1) {
        const int i = __ffs(equal) - 1;
        const uint32_t l = route_logit_key<DT>(p, row, lane * PER + i);
        if (l > mine) {
          mine = l;
          pick = i;
        }
      }
      const uint32_t most = __reduce_max_sync(0xFFFFFFFFu, mine);
      src = __ffs(__ballot_sync(0xFFFFFFFFu, pick >= 0 && mine == most)) - 1;
      if (lane == src) {
        at = lane * PER + pick;
#pragma unroll kUnroll
        for (int i = 0; i < PER; ++i)
          if (i == pick) {
            key[i] = 0;
            sv = s[i];
          }
      }
    } else {
      src = __ffs(__ballot_sync(0xFFFFFFFFu, best == top)) - 1;
      if (lane == src) {
        bool done = false;
#pragma unroll kUnroll
        for (int i = 0; i < PER; ++i)
          if (!done && key[i] == top) {
            done = true;
            key[i] = 0;
            at = lane * PER + i;
            sv = s[i];
          }
      }
    }
    at = __shfl_sync(0xFFFFFFFFu, at, src);
    sv = __shfl_sync(0xFFFFFFFFu, sv, src);
    if (lane == j) { my_id = at; my_w = sv; }
  }
  if (p.renorm) {
    const double t = warp_sum64(my_w);
    my_w = t > 0.0 ? my_w / t : 0.0;
  }
  if (lane < p.k) {
    p.w[row * p.k + lane] = (float)(my_w * (double)p.scale);
    p.ids[row * p.k + lane] = my_id;
  }
  return false;
}

// ONLY_LOGITS: no bias and no top-2 group sums, so logits decide (exactly).
template <int PER, int DT, bool ONLY_LOGITS>
__global__ void __launch_bounds__(32 * kRouteWarps) route_topk_kernel(const RouteParams p) {
  const int64_t row = blockIdx.x * (int64_t)kRouteWarps + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= p.T) return;
  float l[PER];
  {
    using Tp = typename In<DT>::T;
    const Tp* src = reinterpret_cast<const Tp*>(p.logits) + row * p.ld + lane * PER;
    if (p.vec) {
      // E % PER == 0: a lane's piece lies inside the row or past it
      constexpr int kBytes = PER * (int)sizeof(Tp);
      __align__(16) Tp v[PER];
      if (lane * PER < p.E) {
        if constexpr (kBytes >= 16) {
#pragma unroll
          for (int i = 0; i < kBytes / 16; ++i)
            reinterpret_cast<uint4*>(v)[i] = __ldg(reinterpret_cast<const uint4*>(src) + i);
        } else if constexpr (kBytes == 8) {
          *reinterpret_cast<uint2*>(v) = __ldg(reinterpret_cast<const uint2*>(src));
        } else if constexpr (kBytes == 4) {
          *reinterpret_cast<uint32_t*>(v) = __ldg(reinterpret_cast<const uint32_t*>(src));
        } else {
          v[0] = *src;
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) l[i] = In<DT>::to_f(v[i]);
      } else {
#pragma unroll
        for (int i = 0; i < PER; ++i) l[i] = -INFINITY;
      }
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) l[i] = lane * PER + i < p.E ? In<DT>::load(src + i) : -INFINITY;
    }
  }

  // scores
  float s[PER];
  bool bad = false;
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    bad |= l[i] != l[i];
    m = fmaxf(m, l[i]);
  }
  m = order_val(__reduce_max_sync(0xFFFFFFFFu, order_key(m)));
  float smax;
  if (p.sigmoid) {
#pragma unroll
    for (int i = 0; i < PER; ++i) s[i] = __fdividef(1.0f, 1.0f + expf(-l[i]));   // 0 from a divisor of 2^126 on
    smax = 1.0f;
  } else {
    bad |= m == INFINITY;
    const float base = m == -INFINITY ? 0.0f : m;
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      s[i] = expf(l[i] - base);
      t += s[i];
    }
    t = warp_sum(t);
    const float inv = t > 0.0f ? __fdividef(1.0f, t) : 0.0f;
#pragma unroll
    for (int i = 0; i < PER; ++i) s[i] *= inv;
    smax = inv;
  }

  // choice keys
  uint32_t key[PER];
  float cmax = 0.0f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = lane * PER + i;
    float c = l[i];
    if constexpr (!ONLY_LOGITS) {
      const float b = (p.bias && e < p.E) ? __ldg(p.bias + e) : 0.0f;
      c = l[i] == -INFINITY ? -INFINITY : s[i] + b;
      bad |= c != c;
      if (fabsf(c) < INFINITY) cmax = fmaxf(cmax, fabsf(c));
    }
    c += 0.0f;   // -0 and +0 are equal
    key[i] = e < p.E ? order_key(c) : 0u;
  }
  if (__any_sync(0xFFFFFFFFu, bad)) {
    if (lane < p.k) {
      p.w[row * p.k + lane] = __int_as_float(0x7FC00000);
      p.ids[row * p.k + lane] = lane;
    }
    return;
  }
  // How far two f32 choice values may be from the exact ones together. A
  // softmax score: expf 2 ulp, its argument's rounding (|x| 2^-24 exp(x) <=
  // 2^-24 / e), a sum of at most 1024 terms in chains of 37 additions and the
  // quotient: under 3e-6 of the score. A sigmoid: under 1e-6. Then the
  // addition of the bias, 2^-24 of the sum, twice for a group's two terms.
  float tol = 0.0f;
  bool again = false;
  if constexpr (!ONLY_LOGITS) {
    cmax = __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(cmax)));
    tol = (p.sigmoid ? 2e-6f : 6e-6f) * smax + 2.5e-7f * cmax;
  }

  if (p.n_group > 1) {
    const int S = p.E / p.n_group;
    float worth = -INFINITY;
    const int lpg = S / PER;         // lanes per group
    if (S % PER == 0 && (lpg & (lpg - 1)) == 0) {
      // all groups at once: each lane's two largest, then those of the lanes
      // of its group
      uint32_t a = 0, b = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        b = max(b, min(a, key[i]));
        a = max(a, key[i]);
      }
      for (int o = 1; o < lpg; o <<= 1) {
        const uint32_t c = __shfl_xor_sync(0xFFFFFFFFu, a, o), d = __shfl_xor_sync(0xFFFFFFFFu, b, o);
        b = max(max(b, d), min(a, c));
        a = max(a, c);
      }
      float v = order_val(a);
      if (p.top2 && b > kNegInfKey) v += order_val(b);
      worth = __shfl_sync(0xFFFFFFFFu, v, lane * lpg);     // lane g holds group g's
      if (lane >= p.n_group) worth = -INFINITY;
    } else {
      for (int g = 0; g < p.n_group; ++g) {
        uint32_t a = 0, b = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const int e = lane * PER + i;
          if (e >= g * S && e < (g + 1) * S) {
            b = max(b, min(a, key[i]));
            a = max(a, key[i]);
          }
        }
        const uint32_t ga = __reduce_max_sync(0xFFFFFFFFu, a);
        float v = order_val(ga);
        if (p.top2) {
          const int who = __ffs(__ballot_sync(0xFFFFFFFFu, a == ga)) - 1;
          const uint32_t gb = __reduce_max_sync(0xFFFFFFFFu, lane == who ? b : a);
          if (gb > kNegInfKey) v += order_val(gb);
        }
        if (lane == g) worth = v;
      }
    }
    bool near = false;
    const uint32_t keep = keep_groups<float>(worth, p.n_group, p.topk_group, 2.0f * tol, near);
    if (!ONLY_LOGITS) again = near;
    // a lane's experts lie in at most ceil(PER / S) + 1 groups
    int g = lane * PER / S, left = (g + 1) * S - lane * PER;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (lane * PER + i < p.E && !((keep >> g) & 1u)) key[i] = kNegInfKey;
      if (--left == 0) { ++g; left = S; }
    }
  }

  float my_w = 0.0f;
  int my_id = p.E;
  float prev = INFINITY;
  int prev_id = -1;
  for (int j = 0; j < p.k; ++j) {
    uint32_t best = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) best = max(best, key[i]);
    const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, best);
    if (top <= kNegInfKey) break;
    const int src = __ffs(__ballot_sync(0xFFFFFFFFu, best == top)) - 1;
    int at = 0;
    float sv = 0.0f;
    if (lane == src) {
      bool done = false;
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (!done && key[i] == top) {
          done = true;
          key[i] = 0;
          at = lane * PER + i;
          sv = s[i];
        }
    }
    at = __shfl_sync(0xFFFFFFFFu, at, src);
    sv = __shfl_sync(0xFFFFFFFFu, sv, src);
    if constexpr (!ONLY_LOGITS) {
      const float c = order_val(top);
      again |= c == INFINITY;              // there may be more of them
      if (prev - c <= tol && prev_id >= 0) {
        // equal logits and biases: equal choice values, to the lower index
        const float la = route_logit<DT>(p, row, at), lb = route_logit<DT>(p, row, prev_id);
        const float ba = p.bias ? p.bias[at] : 0.0f, bb = p.bias ? p.bias[prev_id] : 0.0f;
        again |= !(la == lb && ba == bb);
      }
      prev = c;
      prev_id = at;
    }
    if (lane == j) { my_id = at; my_w = sv; }
  }
  if constexpr (!ONLY_LOGITS) {
    // is any expert left that may be better than the last one taken? (Not only
    // the next: behind several equal ones f32 may hide a better one.)
    uint32_t close = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) close |= (uint32_t)(key[i] > kNegInfKey && prev - order_val(key[i]) <= tol) << i;
    if (prev_id >= 0 && __any_sync(0xFFFFFFFFu, close)) {
      const float la = route_logit<DT>(p, row, prev_id), ba = p.bias ? p.bias[prev_id] : 0.0f;
      bool differs = false;
      for (; close; close &= close - 1) {
        const int e = lane * PER + __ffs(close) - 1;
        differs |= !(route_logit<DT>(p, row, e) == la && (p.bias ? p.bias[e] : 0.0f) == ba);
      }
      again |= __any_sync(0xFFFFFFFFu, differs);
    }
  }
  // scores that f32 holds with fewer bits, or not at all
  const uint32_t used = __ballot_sync(0xFFFFFFFFu, my_id < p.E);
  const float sum = warp_sum(my_w);
  again |= used != 0 && sum < 1e-30f;
  if (again) {
    if (route_row64<PER, DT, ONLY_LOGITS, false>(p, row))
      if constexpr (!ONLY_LOGITS) route_row64<PER, DT, ONLY_LOGITS, true>(p, row);
    return;
  }
  if (p.renorm) my_w = sum > 0.0f ? my_w / sum : 0.0f;
  if (lane < p.k) {
    p.w[row * p.k + lane] = my_w * p.scale;
    p.ids[row * p.k + lane] = my_id;
  }
}

// ---------------------------------------------------------------- many rows
// One thread per row, for 16-bit logits that alone decide (no bias, no
// groups) and k <= 8. A logit and its index make one 32-bit key that orders
// as they do, so a comparison of two candidates is one max and one min: eight
// keys at a time are sorted (19 of them) and merged into the best eight so
// far (8 + 12), 35 instructions per row and warp lane at 128 experts where
// the warp above takes some 800. The rows are staged through shared memory,
// read with whole lines.
constexpr int kRouteRowThreads = 128;
// From how many rows, of bf16 and k = 8 (us, the warp kernel / this one):
// 64 experts 2048 rows 6.2 / 6.2, 8192 rows 10.3 / 6.2; 128 experts 2048 rows
// 6.2 / 8.3, 4096 rows 8.3 / 8.3, 65536 rows 51 / 17; 256 experts 4096 rows
// 10.0 / 12.5, 8192 rows 14.4 / 12.5; 512 experts 8192 rows 20.9 / 20.6, 16384
// rows 37 / 21. With fewer rows its threads, one per row, do not fill the SMs.
constexpr int64_t kRouteRowsFrom = 4096, kRouteRowsPerExpert = 32;

__device__ __forceinline__ void key_pair(uint32_t& a, uint32_t& b) {
  const uint32_t t = max(a, b);
  b = min(a, b);
  a = t;
}
__device__ __forceinline__ void sort8(uint32_t (&v)[8]) {      // descending
  key_pair(v[0], v[1]); key_pair(v[2], v[3]); key_pair(v[4], v[5]); key_pair(v[6], v[7]);
  key_pair(v[0], v[2]); key_pair(v[1], v[3]); key_pair(v[4], v[6]); key_pair(v[5], v[7]);
  key_pair(v[1], v[2]); key_pair(v[5], v[6]); key_pair(v[0], v[4]); key_pair(v[3], v[7]);
  key_pair(v[1], v[5]); key_pair(v[2], v[6]);
  key_pair(v[1], v[4]); key_pair(v[3], v[6]);
  key_pair(v[2], v[4]); key_pair(v[3], v[5]);
  key_pair(v[3], v[4]);
}

template <int DT>
__global__ void __launch_bounds__(kRouteRowThreads) route_rows_kernel(const RouteParams p) {
  using Tp = typename In<DT>::T;
  extern __shared__ __align__(16) uint8_t rows[];
  const int64_t row0 = blockIdx.x * (int64_t)kRouteRowThreads;
  const int n = (int)min((int64_t)kRouteRowThreads, p.T - row0);
  const int chunks = p.E / 8, pitch = 2 * p.E + 16;       // 16 bytes more: 8 rows, 8 different bank groups
  for (int i = threadIdx.x; i < n * chunks; i += kRouteRowThreads) {
    const int r = i / chunks, c = i - r * chunks;
    *reinterpret_cast<uint4*>(rows + r * pitch + 16 * c) =
        __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const Tp*>(p.logits) + (row0 + r) * p.ld) + c);
  }
  __syncthreads();
  if ((int)threadIdx.x >= n) return;
  const uint8_t* mine = rows + threadIdx.x * pitch;
  constexpr uint32_t kInf = DT == AEOQ_BF16 ? 0x7F80u : 0x7C00u;
  uint32_t best[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
  uint32_t most = 0;      // largest magnitude pattern: NaN above infinity
  for (int c = 0; c < chunks; ++c) {
    const uint4 u = *reinterpret_cast<const uint4*>(mine + 16 * c);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    uint32_t v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t b = (w[i >> 1] >> (16 * (i & 1))) & 0xFFFFu;
      most = max(most, b & 0x7FFFu);
      b = b == 0x8000u ? 0u : b;                                  // -0 and +0 are equal
      b = (b & 0x8000u) ? b ^ 0xFFFFu : b | 0x8000u;
      v[i] = (b << 16) | (0xFFFFu - (uint32_t)(8 * c + i));         // equal logits: the lower index first
    }
    sort8(v);
#pragma unroll
    for (int i = 0; i < 8; ++i) best[i] = max(best[i], v[7 - i]);
#pragma unroll
    for (int d = 4; d >= 1; d >>= 1)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (!(i & d)) key_pair(best[i], best[i + d]);
  }
  const int64_t row = row0 + threadIdx.x;
  float* wo = p.w + row * p.k;
  int64_t* io = p.ids + row * p.k;
  const auto logit = [&](uint32_t key) {
    const uint32_t b = key >> 16;
    return In<DT>::key_to_f((b & 0x8000u) ? b & 0x7FFFu : b ^ 0xFFFFu);
  };
  const float top = logit(best[0]);
  if (most > kInf || (!p.sigmoid && top == INFINITY)) {
    for (int j = 0; j < p.k; ++j) {
      wo[j] = __int_as_float(0x7FC00000);
      io[j] = j;
    }
    return;
  }
  float s[8], sum = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float l = logit(best[j]);
    s[j] = 0.0f;
    if (j < p.k && l > -INFINITY) s[j] = p.sigmoid ? __fdividef(1.0f, 1.0f + expf(-l)) : expf(l - top);
    sum += s[j];
  }
  if (p.sigmoid && top > -INFINITY && sum < 1e-30f) {      // f32 has lost them
    double d[8], t = 0.0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float l = logit(best[j]);
      d[j] = j < p.k && l > -INFINITY ? 1.0 / (1.0 + exp(-(double)l)) : 0.0;
      t += d[j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] = (float)(p.renorm ? (t > 0.0 ? d[j] / t : 0.0) : d[j]);
    sum = 1.0f;
  } else if (p.renorm) {
    const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] *= inv;
  } else if (!p.sigmoid && top > -INFINITY) {
    float t = 0.0f;
    for (int c = 0; c < chunks; ++c) {
      const uint4 u = *reinterpret_cast<const uint4*>(mine + 16 * c);
      const Tp* e = reinterpret_cast<const Tp*>(&u);
      float part = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) part += expf(In<DT>::to_f(e[i]) - top);
      t += part;
    }
    const float inv = 1.0f / t;
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] *= inv;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (j >= p.k) break;
    const bool none = logit(best[j]) == -INFINITY;
    wo[j] = none ? 0.0f : s[j] * p.scale;
    io[j] = none ? p.E : (int64_t)(0xFFFFu - (best[j] & 0xFFFFu));
  }
}

template <int DT>
static int launch_route_rows(const RouteParams& p, cudaStream_t st) {
  const size_t bytes = (size_t)kRouteRowThreads * (2 * p.E + 16);
  const int rc = func_smem_attr((const void*)route_rows_kernel<DT>, bytes, -1, "route_rows");
  if (rc) return rc;
  const unsigned blocks = (unsigned)((p.T + kRouteRowThreads - 1) / kRouteRowThreads);
  route_rows_kernel<DT><<<blocks, kRouteRowThreads, bytes, st>>>(p);
  return check_launch("route_rows_kernel");
}

template <int PER, int DT>
static int launch_route(const RouteParams& p, cudaStream_t st) {
  const unsigned blocks = (unsigned)((p.T + kRouteWarps - 1) / kRouteWarps);
  if (!p.bias && !(p.n_group > 1 && p.top2))
    route_topk_kernel<PER, DT, true><<<blocks, 32 * kRouteWarps, 0, st>>>(p);
  else
    route_topk_kernel<PER, DT, false><<<blocks, 32 * kRouteWarps, 0, st>>>(p);
  return check_launch("route_topk_kernel");
}

template <int DT>
static int dispatch_route(RouteParams p, cudaStream_t st) {
  int per = 1;
  while (per * 32 < p.E) per *= 2;
  const int bytes = per * (int)sizeof(typename In<DT>::T), width = std::min(bytes, 16);
  p.vec = p.E % per == 0 && (uintptr_t)p.logits % width == 0 &&
          (p.ld * (int64_t)sizeof(typename In<DT>::T)) % width == 0;
  if constexpr (DT != AEOQ_F32) {
    const bool logits_alone = !p.bias && p.n_group == 1;
    if (logits_alone && p.k <= 8 && p.E >= 8 && p.E <= 512 && p.E % 8 == 0 && (uintptr_t)p.logits % 16 == 0 &&
        (p.ld * 2) % 16 == 0 && p.T >= std::max(kRouteRowsFrom, kRouteRowsPerExpert * p.E))
      return launch_route_rows<DT>(p, st);
  }
  switch (per) {
    case 1: return launch_route<1, DT>(p, st);
    case 2: return launch_route<2, DT>(p, st);
    case 4: return launch_route<4, DT>(p, st);
    case 8: return launch_route<8, DT>(p, st);
    case 16: return launch_route<16, DT>(p, st);
    default: return launch_route<32, DT>(p, st);
  }
}

}  // namespace aeoq

using namespace aeoq;

extern "C" int aeoq_route_topk(const void* logits, int dtype, int64_t ld, int64_t T, int64_t num_experts, int64_t k,
                               int score, const float* bias, int64_t n_group, int64_t topk_group, int group_score,
                               int renormalize, float scale, float* weights, int64_t* ids, void* stream) {
  AEOQ_REQUIRE(num_experts >= 1 && num_experts <= kRouteMaxExperts, AEOQ_ERR_INVALID,
               "route_topk: num_experts (%lld) must be in [1, %d]", (long long)num_experts, kRouteMaxExperts);
  AEOQ_REQUIRE(k >= 1 && k <= std::min<int64_t>(num_experts, kRouteMaxK), AEOQ_ERR_INVALID,
               "route_topk: k (%lld) must be in [1, min(num_experts, %d)]", (long long)k, kRouteMaxK);
  AEOQ_REQUIRE(n_group >= 1 && n_group <= kRouteMaxGroups && num_experts % n_group == 0, AEOQ_ERR_INVALID,
               "route_topk: n_group (%lld) must be in [1, %d] and divide num_experts (%lld)", (long long)n_group,
               kRouteMaxGroups, (long long)num_experts);
  AEOQ_REQUIRE(topk_group >= 1 && topk_group <= n_group, AEOQ_ERR_INVALID,
               "route_topk: topk_group (%lld) must be in [1, n_group]", (long long)topk_group);
  AEOQ_REQUIRE((score == AEOQ_SCORE_SOFTMAX || score == AEOQ_SCORE_SIGMOID) &&
                   (group_score == AEOQ_GROUP_MAX || group_score == AEOQ_GROUP_TOP2),
               AEOQ_ERR_INVALID, "route_topk: bad score (%d) or group score (%d)", score, group_score);
  AEOQ_REQUIRE(T >= 0 && ld >= num_experts, AEOQ_ERR_INVALID, "route_topk: bad shape");
  AEOQ_REQUIRE(T <= 8LL * 1024 * 1024 * 1024, AEOQ_ERR_INVALID, "route_topk: too many tokens");
  if (T == 0) return AEOQ_OK;
  AEOQ_REQUIRE(logits && weights && ids, AEOQ_ERR_INVALID, "route_topk: null pointer");
  RouteParams p{};
  p.logits = logits;
  p.ld = ld;
  p.T = T;
  p.E = (int)num_experts;
  p.k = (int)k;
  p.bias = bias;
  p.n_group = (int)(topk_group == n_group ? 1 : n_group);   // every group stays: none to choose
  p.topk_group = (int)topk_group;
  p.sigmoid = score == AEOQ_SCORE_SIGMOID;
  p.top2 = group_score == AEOQ_GROUP_TOP2;
  p.renorm = renormalize != 0;
  p.scale = scale;
  p.w = weights;
  p.ids = ids;
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case AEOQ_BF16: return dispatch_route<AEOQ_BF16>(p, st);
    case AEOQ_F16: return dispatch_route<AEOQ_F16>(p, st);
    case AEOQ_F32: return dispatch_route<AEOQ_F32>(p, st);
  }
  return set_error(AEOQ_ERR_INVALID, "route_topk: unsupported dtype %d", dtype);
}
