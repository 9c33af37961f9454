// Balanced routing: top-k of the experts by score plus a per-expert bias
// that steers the load, with weights from the unbiased scores, and the
// gradient of those weights with respect to the router logits.
//
//   s_e = sigmoid(l_e)   or   exp(l_e - max l) / sum_e' exp(l_e' - max l)
//   c_e = s_e + bias_e
//   group value = sum of the group's two largest c (or its largest)
//   kept  = the topk_group groups of largest value
//   chosen = the top_k experts of largest c in the kept groups, in order
//   w_j = scale * s_j            or, renormalised, scale * s_j / sum_i s_i
// Ties go to the lower index. Unlike a top-k by logit, the order of c cannot
// be read off the logits, and two c that differ by less than a 32-bit
// rounding must still come out in their true order for the ids to be a
// function of the inputs alone. So each row is first selected in 32 bits; a
// comparison that decided the result by less than the error bound of the
// 32-bit scores (and that is not between equal logits with equal biases,
// a true tie) sends the warp through the same code in 64 bits.
//
// One warp per token, the row in registers (lane l holds the PL experts from l PL
// on). Where a group is the experts of a power of two of lanes, its value is
// reduced among them; other groups' from shared memory, by 32 / G lanes per group
// at once (8192 x 256 in 8 groups 13.7 us the first way, 15.3 the second, with lane
// l holding experts l, l + 32, ...). What bounds it: instruction issue and
// latency, not its T*E*4 bytes (about 1090 instructions per token of 256 experts
// in 8 groups). One B200: 8192 x 256 in 8 groups, top 8, 13.5 us; 4096 x 128 7.3
// us; 16384 x 384 35 us; one token of 256 3.4 us.
#include <atomic>
#include <type_traits>

#include "common.cuh"

namespace ksw {
namespace {

// Warps (tokens) per block; 1 and 2 measured the same from 1 to 16384 tokens.
constexpr int kWarps = 4;

struct BalanceParams {
  const void* logits;
  const float* bias;  // may be null
  int64_t T;
  int E, k, G, EG, kept;
  uint32_t eg_magic;  // ceil(2^22 / EG): e / EG = (e * eg_magic) >> 22 for e < 1024, EG <= 1024
  // lanes that reduce a group's value, a power of two, and its logarithm: those
  // that hold its experts (in_lanes), else as many as 32 lanes allow
  int lanes_per_group, group_shift, in_lanes;
  int vec, vec_bias;  // a lane's logits and biases may be loaded as 16-byte vectors
  int softmax, top2, renorm;
  float scale;
  void* weights;
  int w_dtype;
  void* ids;
  int ids64;
  int32_t* load;  // may be null
};

__device__ __forceinline__ uint32_t group_of(const BalanceParams& p, int e) {
  return (uint32_t(e) * p.eg_magic) >> 22;
}

// Largest value of a 32-bit key over the warp.
__device__ __forceinline__ uint32_t redux_max(uint32_t v) {
  return __reduce_max_sync(0xffffffffu, v);
}
// Order-preserving map of floats to unsigned integers; 0 is below all of them.
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t u = __float_as_uint(v);
  return u ^ (uint32_t(int32_t(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

template <typename R>
__device__ __forceinline__ R warp_sum(R v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// The 32-bit scores that the choice is first made by: fast exponentials and
// reciprocals, whose errors the choice allows for. The PTX manual gives 2^-22 for
// ex2.approx and 1 ulp for rcp.approx; the argument's product with log2(e) is
// off by half an ulp of itself, |x| * 2^-24 in the result's relative error, and
// as much again through the constant.
__device__ __forceinline__ float score_exp(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
  return y;
}
__device__ __forceinline__ double score_exp(double x) { return exp(x); }
__device__ __forceinline__ float score_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ double score_rcp(double x) { return 1.0 / x; }

// Error bound of one 32-bit score, per unit of the row's largest, in ulp (2^-23);
// exp(x) is off by 2 + |x|. Sigmoid: exp's error counts (1 - s) times; s (1 - s)
// |x| is under 0.23 for positive logits, and for negative ones s is e^l to first
// order, so that 2 + |l| counts at the largest logit (below it s falls faster
// than |l| grows); the add and the reciprocal 1.5. Softmax: e^-d (2 + d) <= 2 for
// exp, the difference l - max 0.2, the reciprocal and the product 1.5, and the
// error of the sum, which the terms at distance d share in by their weight: their
// mean d is at most ln 1024 < 7, so 9 for the terms, and half an ulp for each of
// the PL + 4 additions. To this the caller adds 2^-126: results below it are flushed
// to 0.
template <int PL>
__device__ __forceinline__ float score_ulps(int softmax, float mx) {
  return softmax ? 16.0f + 0.5f * (PL + 4) : 6.0f + 1.2f * fmaxf(-mx, 0.0f);
}

// A lane's PL values of a row of E: whole vectors where the caller says so (E is
// then a multiple of PL), `rest` behind the row's end.
template <int PL, typename T>
__device__ __forceinline__ void load_lane(const T* row, int E, int lane, bool vec, float rest,
                                          float (&v)[PL]) {
  constexpr int kBytes = PL * int(sizeof(T));
  if constexpr (kBytes % 16 == 0) {
    if (vec) {
      const uint4* at = reinterpret_cast<const uint4*>(row + lane * PL);
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i) {
        const uint4 w = lane * PL < E ? __ldg(at + i) : make_uint4(0, 0, 0, 0);
        const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
        for (int j = 0; j < 16 / int(sizeof(T)); ++j)
          v[i * (16 / int(sizeof(T))) + j] = lane * PL < E ? to_f32(e[j]) : rest;
      }
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < PL; ++j) {
    const int e = lane * PL + j;
    v[j] = e < E ? to_f32(row[e]) : rest;
  }
}

// c of the row's experts, lane l's j-th being expert l PL + j, -inf behind the
// last. `mx` is the row's largest logit; a NaN ranks last. `smax` returns the
// largest score.
template <typename R, int PL, typename Tin>
__device__ __forceinline__ void biased_scores(const BalanceParams& p, const float (&l)[PL],
                                              float mx, int lane, R (&c)[PL], R& smax) {
  const R rmx = mx == -INFINITY ? R(0) : R(mx);
  float b[PL];
  if (p.bias != nullptr) {
    load_lane<PL>(p.bias, p.E, lane, p.vec_bias, -INFINITY, b);
  } else {
#pragma unroll
    for (int j = 0; j < PL; ++j) b[j] = lane * PL + j < p.E ? 0.0f : -INFINITY;
  }
  if (p.softmax) {
    R sum = R(0);
#pragma unroll
    for (int j = 0; j < PL; ++j) {
      c[j] = score_exp(R(l[j]) - rmx);
      if (lane * PL + j < p.E) sum += c[j];
    }
    sum = warp_sum(sum);
    const bool none = mx == -INFINITY;  // no expert has a score: all 0
    smax = none ? R(0) : score_rcp(sum);
#pragma unroll
    for (int j = 0; j < PL; ++j) c[j] = none ? R(0) : c[j] * smax;
  } else {
#pragma unroll
    for (int j = 0; j < PL; ++j) c[j] = score_rcp(R(1) + score_exp(-R(l[j])));
    smax = mx == -INFINITY ? R(0) : score_rcp(R(1) + score_exp(-rmx));
  }
#pragma unroll
  for (int j = 0; j < PL; ++j) {
    const R v = c[j] + R(b[j]);
    c[j] = v != v ? R(-INFINITY) : v;
  }
}

// Two largest of (a >= b) and v.
__device__ __forceinline__ void top_two(float v, float& a, float& b) {
  b = fmaxf(b, fminf(a, v));
  a = fmaxf(a, v);
}
__device__ __forceinline__ void top_two(double v, double& a, double& b) {
  b = fmax(b, fmin(a, v));
  a = fmax(a, v);
}

// Bit g * lanes_per_group: group g is kept. Groups are compared by half their
// value, which stays in range where two of the type's lowest numbers are added.
// In 32 bits half a value is off by `slack` for its scores, and by 2^-22 of its
// terms' (halved) magnitudes, which may cancel while their roundings do not: half
// an ulp of each, lost when its bias was added, as much at most for their sum, and
// twice that. Sets `close` when a group left out may lie above any of those kept:
// each has a bound of its own, so the one in doubt need not be the last one kept.
template <typename R, int PL>
__device__ __forceinline__ uint32_t kept_groups(const BalanceParams& p, const R (&c)[PL],
                                                int lane, R* scratch, float slack, bool& close) {
  const int per = p.lanes_per_group;
  const int g = lane >> p.group_shift, sub = lane & (per - 1);
  R a = R(-INFINITY), b = R(-INFINITY);  // the two largest, a >= b
  if (p.in_lanes) {
#pragma unroll
    for (int j = 0; j < PL; ++j) top_two(c[j], a, b);
  } else {
    // position e + group keeps lanes of different groups on different banks
    __syncwarp();
#pragma unroll
    for (int j = 0; j < PL; ++j) {
      const int e = lane * PL + j;
      if (e < p.E) scratch[e + group_of(p, e)] = c[j];
    }
    __syncwarp();
    if (g < p.G) {
      const R* at = scratch + g * (p.EG + 1);
#pragma unroll 4
      for (int i = sub; i < p.EG; i += per) top_two(at[i], a, b);
    }
  }
  for (int o = per >> 1; o > 0; o >>= 1) {
    const R oa = __shfl_xor_sync(0xffffffffu, a, o);
    const R ob = __shfl_xor_sync(0xffffffffu, b, o);
    top_two(oa, a, b);
    top_two(ob, a, b);
  }
  if (!p.top2 || p.EG == 1) b = R(0);  // a group of one has no second
  const R ha = R(0.5) * a, hb = R(0.5) * b;
  R value = ha + hb;
  if (value != value) value = R(-INFINITY);  // +inf and -inf in one group
  // a group's rank: how many come before it
  int rank = 0;
  for (int h = 0; h < p.G; ++h) {
    const R o = __shfl_sync(0xffffffffu, value, h * per);
    rank += o > value || (o == value && h < g);
  }
  const bool mine = g < p.G && sub == 0;
  const bool keep = mine && rank < p.kept;
  if constexpr (std::is_same<R, float>::value) {
    // infinite values are exact. An infinite kept one's lower bound is NaN, whose key
    // is above all others, or -inf; one left out has a NaN for its upper bound then
    const float e = slack + 0x1p-22f * (fabsf(ha) + fabsf(hb));
    const uint32_t low = __reduce_min_sync(0xffffffffu, keep ? order_key(value - e) : UINT32_MAX);
    close = mine && !keep && value + e >= key_value(low);
  }
  return __ballot_sync(0xffffffffu, keep);
}
// Bit j: this lane's expert j exists and its group is kept.
template <int PL>
__device__ __forceinline__ uint32_t open_experts(const BalanceParams& p, uint32_t kept, int lane) {
  const int first = lane * PL;
  uint32_t open = first + PL <= p.E ? 0xffffffffu : first < p.E ? (1u << (p.E - first)) - 1 : 0u;
  if (p.in_lanes) {
    if (!((kept >> (lane & ~(p.lanes_per_group - 1))) & 1u)) open = 0;
  } else if (p.G > 1) {
#pragma unroll
    for (int j = 0; j < PL; ++j)
      if (!((kept >> (group_of(p, min(first + j, p.E - 1)) << p.group_shift)) & 1u))
        open &= ~(1u << j);
  }
  return open;
}

// Puts n <= 32 candidates (lane i < n: expert `e`) in their order in 64 bits and
// returns the first k, lane s the s-th. `list` holds 32 indexes for this warp.
// Out of the kernel's body, whose registers it would double: few rows need it.
template <typename Tin>
__device__ __noinline__ int order_exact(const BalanceParams& p, const Tin* row, float mx, int lane,
                                        int n, int e, int* list) {
  double c = -INFINITY;
  double sum = 0.0;
  const bool none = mx == -INFINITY;
  if (p.softmax && !none) {
    for (int i = lane; i < p.E; i += 32) sum += exp(double(to_f32(row[i])) - double(mx));
    sum = warp_sum(sum);
  }
  if (lane < n) {
    const double l = to_f32(row[e]);
    const double s = p.softmax ? (none ? 0.0 : exp(l - double(mx)) / sum) : 1.0 / (1.0 + exp(-l));
    c = s + (p.bias != nullptr ? double(__ldg(p.bias + e)) : 0.0);
    if (c != c) c = -INFINITY;
  }
  int rank = 0;
  for (int h = 0; h < n; ++h) {
    const double oc = __shfl_sync(0xffffffffu, c, h);
    const int oe = __shfl_sync(0xffffffffu, e, h);
    rank += oc > c || (oc == c && oe < e);
  }
  if (lane < n) list[rank] = e;
  __syncwarp();
  const int sel = lane < p.k ? list[lane] : 0;
  __syncwarp();
  return sel;
}

// c of the row in 64 bits, from its logits in memory.
template <int PL, typename Tin>
__device__ __forceinline__ void exact_scores(const BalanceParams& p, const Tin* row, float mx,
                                             int lane, double (&c)[PL]) {
  float l[PL];
  load_lane<PL>(row, p.E, lane, p.vec, -INFINITY, l);
  double smax;
  biased_scores<double, PL, Tin>(p, l, mx, lane, c, smax);
}

// The groups kept, in 64 bits (kept_groups' mask).
template <int PL, typename Tin>
__device__ __noinline__ uint32_t kept_exact(const BalanceParams& p, const Tin* row, float mx,
                                            int lane, double* scratch) {
  double c[PL];
  exact_scores<PL>(p, row, mx, lane, c);
  bool close = false;
  return kept_groups(p, c, lane, scratch, 0.0f, close);
}

// The row's experts in 64 bits, groups included: lane s < k returns the s-th.
template <int PL, typename Tin>
__device__ __noinline__ int select_exact(const BalanceParams& p, const Tin* row, float mx,
                                         int lane, double* scratch) {
  double c[PL];
  exact_scores<PL>(p, row, mx, lane, c);
  uint32_t kept = 0xffffffffu;
  bool close = false;
  if (p.G > 1) kept = kept_groups(p, c, lane, scratch, 0.0f, close);
  uint32_t open = open_experts<PL>(p, kept, lane);
  int sel = 0;
  for (int s = 0; s < p.k; ++s) {
    double v = -INFINITY;
    int i = INT32_MAX;
#pragma unroll
    for (int j = 0; j < PL; ++j)
      if (((open >> j) & 1u) && (i == INT32_MAX || c[j] > v)) {
        v = c[j];
        i = lane * PL + j;
      }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const double ov = __shfl_xor_sync(0xffffffffu, v, o);
      const int oi = __shfl_xor_sync(0xffffffffu, i, o);
      if (oi != INT32_MAX && (i == INT32_MAX || ov > v || (ov == v && oi < i))) {
        v = ov;
        i = oi;
      }
    }
    if (i / PL == lane) open &= ~(1u << (i % PL));
    if (lane == s) sel = i;
  }
  return sel;
}

// Whether two experts tie in truth: equal logits and equal biases.
template <typename Tin>
__device__ __forceinline__ bool true_tie(const BalanceParams& p, const Tin* row, int a, int b) {
  return to_f32(row[a]) == to_f32(row[b]) &&
         (p.bias == nullptr || __ldg(p.bias + a) == __ldg(p.bias + b));
}

// The same in 32 bits; a row some of whose comparisons were too close to trust
// goes on in 64: the groups where one's place was in doubt, then the chosen and
// those within the tolerance of the last one. The values are held as ordered
// unsigned keys whose low bits give way to the lane's index of the expert (PL - 1
// - j, so that ties go to the lower one), 0 for one that cannot be chosen. Each
// lane sorts its keys; a pick is the largest of the lanes' first keys, their low
// bits apart, popped in the lowest lane that has it.
template <int PL, typename Tin>
__device__ __forceinline__ int select_row(const BalanceParams& p, const Tin* row,
                                          const float (&l)[PL], float mx, int lane,
                                          double* scratch, int* list) {
  float c[PL], smax;
  biased_scores<float, PL, Tin>(p, l, mx, lane, c, smax);
  // of a difference of two c: both scores, the rounding of both sums with the
  // bias and the bits cut off both keys; twice that, since it is itself rounded
  const float scores = 2.0f * 2.0f * (score_ulps<PL>(p.softmax, mx) * 0x1p-23f * smax + 0x1p-126f);
  auto tol = [&](float v) { return scores + 2.0f * 2.0f * (PL + 0.5f) * 0x1p-23f * fabsf(v); };
  uint32_t kept = 0xffffffffu;
  if (p.G > 1) {
    // half a value has the error of one score
    bool close = false;
    kept = kept_groups(p, c, lane, reinterpret_cast<float*>(scratch), 0.5f * scores, close);
    if (__any_sync(0xffffffffu, close)) kept = kept_exact<PL>(p, row, mx, lane, scratch);
  }
  constexpr uint32_t kLow = PL - 1;
  uint32_t key[PL];
  const uint32_t open = open_experts<PL>(p, kept, lane);
#pragma unroll
  for (int j = 0; j < PL; ++j)
    key[j] = (open >> j) & 1u ? (order_key(c[j]) & ~kLow) | (kLow - j) : 0u;
  // bitonic sort, descending
#pragma unroll
  for (int w = 2; w <= PL; w <<= 1)
#pragma unroll
    for (int d = w >> 1; d > 0; d >>= 1)
#pragma unroll
      for (int j = 0; j < PL; ++j)
        if ((j ^ d) > j) {
          const uint32_t lo = min(key[j], key[j ^ d]), hi = max(key[j], key[j ^ d]);
          const bool down = (j & w) == 0;
          key[j] = down ? hi : lo;
          key[j ^ d] = down ? lo : hi;
        }
  int sel = 0, last_i = 0;
  float last = 0.0f;
  bool close = false;
  for (int s = 0; s < p.k; ++s) {
    const uint32_t top = key[0] & ~kLow;
    const uint32_t best = redux_max(top);
    const int src = __ffs(__ballot_sync(0xffffffffu, top == best)) - 1;
    const int i = src * PL + int(kLow - (__shfl_sync(0xffffffffu, key[0], src) & kLow));
    if (lane == s) sel = i;
#pragma unroll
    for (int j = 0; j < PL; ++j) key[j] = lane != src ? key[j] : j + 1 < PL ? key[j + 1] : 0u;
    const float v = key_value(best);
    if (s > 0 && last - v <= tol(last) && !true_tie(p, row, last_i, i)) close = true;
    last = v;
    last_i = i;
  }
  // the experts left out must be clear of the last one chosen
  if (last > -INFINITY) {
    const uint32_t bar = order_key(last - tol(last)) & ~kLow;
    bool near = false;
    if (key[0] >= bar) {
#pragma unroll
      for (int j = 0; j < PL; ++j)
        near |= key[j] >= bar && key[j] != 0u &&
                !true_tie(p, row, last_i, lane * PL + int(kLow - (key[j] & kLow)));
    }
    if (__any_sync(0xffffffffu, near) || close) {
      int n = p.k;
      if (lane < p.k) list[lane] = sel;
#pragma unroll
      for (int j = 0; j < PL; ++j) {
        const bool in = key[j] >= bar && key[j] != 0u;
        const uint32_t who = __ballot_sync(0xffffffffu, in);
        const int at = n + __popc(who & lanemask_lt());
        if (in && at < 32) list[at] = lane * PL + int(kLow - (key[j] & kLow));
        n += __popc(who);
      }
      __syncwarp();
      const int e = list[lane];
      __syncwarp();
      return n <= 32 ? order_exact(p, row, mx, lane, n, e, list)
                     : select_exact<PL>(p, row, mx, lane, scratch);
    }
  } else if (close) {
    return select_exact<PL>(p, row, mx, lane, scratch);
  }
  return sel;
}

// 64 registers for up to 256 experts (8192 x 256 13.4 us against 14.0 with 80). The
// parameters stay in constant memory, where the functions out of line read them
// too (with a copy in each thread's local memory 8192 x 256 takes 14.1 us, 16384 x
// 384 38.5 instead of 34.8).
template <int PL, typename Tin>
__global__ void __launch_bounds__(32 * kWarps, PL <= 8 ? 8 : 4)
    balanced_topk_kernel(const __grid_constant__ BalanceParams p) {
  extern __shared__ double s_scratch[];
  __shared__ int s_list[kWarps][32];
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  double* scratch = s_scratch + (p.G > 1 && !p.in_lanes ? warp * (p.E + p.G) : 0);
  for (int64_t t = int64_t(blockIdx.x) * kWarps + warp; t < p.T;
       t += int64_t(gridDim.x) * kWarps) {
    const Tin* row = static_cast<const Tin*>(p.logits) + t * p.E;
    float l[PL];
    load_lane<PL>(row, p.E, lane, p.vec, -INFINITY, l);
    float mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < PL; ++j) mx = fmaxf(mx, l[j]);
    mx = warp_max(mx);
    const int sel = select_row<PL>(p, row, l, mx, lane, scratch, s_list[warp]);

    // weights of the chosen: lane s < k has the s-th
    const bool mine = lane < p.k;
    const float ls = mine ? to_f32(row[sel]) : -INFINITY;
    float s;
    if (p.softmax) {
      // renormalised over the chosen, the softmax needs the chosen logits only
      const float top = p.renorm ? warp_max(ls) : mx;
      s = ls == -INFINITY ? 0.0f : expf(ls - top);
      if (!p.renorm) {
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < PL; ++j)
          if (l[j] != -INFINITY) sum += expf(l[j] - mx);
        sum = warp_sum(sum);
        s = sum == 0.0f ? 0.0f : s / sum;  // a row of -inf alone has no scores
      }
    } else {
      s = mine ? 1.0f / (1.0f + expf(-ls)) : 0.0f;
    }
    float w = s;
    if (p.renorm) {
      const float total = warp_sum(s);
      w = total == 0.0f ? 0.0f : s / total;  // chosen scores that all vanish: no weight
    }
    w *= p.scale;
    if (mine) {
      const int64_t at = t * p.k + lane;
      if (p.w_dtype == MOE_DTYPE_F32)
        static_cast<float*>(p.weights)[at] = w;
      else if (p.w_dtype == MOE_DTYPE_BF16)
        static_cast<__nv_bfloat16*>(p.weights)[at] = from_f32<__nv_bfloat16>(w);
      else
        static_cast<__half*>(p.weights)[at] = from_f32<__half>(w);
      if (p.ids64)
        static_cast<int64_t*>(p.ids)[at] = sel;
      else
        static_cast<int32_t*>(p.ids)[at] = sel;
      // integer adds: the counts do not depend on their order
      if (p.load != nullptr) atomicAdd(p.load + sel, 1);
    }
  }
}

// ---------------------------------------------------------------------------
// Backward: the ids are constants, w_j = scale * s_j [/ sum_i s_i]. With g_j =
// scale * dL/dw_j, p_j = s_j / sum_i s_i over the chosen and gm = sum_i g_i p_i:
//   sigmoid, renormalised: dl_j = (g_j - gm) p_j (1 - s_j), 0 elsewhere
//   sigmoid:               dl_j = g_j s_j (1 - s_j),        0 elsewhere
//   softmax, renormalised: dl_j = (g_j - gm) p_j,           0 elsewhere
//                          (p is the softmax over the chosen alone)
//   softmax:               dl_e = s_e (g_e - sum_i g_i s_i), g_e = 0 elsewhere
// One warp per token: it fills the row, then lane j < k stores expert j's
// entry. Bound by the T*E*b bytes it writes (and reads, for the last form); at
// 4096 x 128 bf16 it takes 3.1 us (4.3 us in the last form), a fraction of what the
// autograd engine takes to call it.
// ---------------------------------------------------------------------------

struct BalanceGradParams {
  const void* logits;
  const void* ids;
  int ids64;
  const float* grad_weights;
  int64_t T;
  int E, k, softmax, renorm;
  float scale;
  void* grad_logits;
};

template <typename Tin>
__global__ void __launch_bounds__(32 * kWarps)
    balanced_topk_grad_kernel(const BalanceGradParams p) {
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kVec = 16 / int(sizeof(Tin));
  const bool vec = p.E % kVec == 0;  // every row starts on a 16-byte boundary
  for (int64_t t = int64_t(blockIdx.x) * kWarps + warp; t < p.T;
       t += int64_t(gridDim.x) * kWarps) {
    const Tin* row = static_cast<const Tin*>(p.logits) + t * p.E;
    Tin* out = static_cast<Tin*>(p.grad_logits) + t * p.E;
    const bool mine = lane < p.k;
    const int64_t at = t * p.k + lane;
    int64_t id = -1;
    if (mine)
      id = p.ids64 ? static_cast<const int64_t*>(p.ids)[at]
                   : static_cast<const int32_t*>(p.ids)[at];
    const bool valid = id >= 0 && id < p.E;  // an id out of range has no gradient
    const int e = valid ? int(id) : 0;
    const float l = valid ? to_f32(row[e]) : -INFINITY;
    const float g = valid ? p.scale * p.grad_weights[at] : 0.0f;
    float d = 0.0f;     // this lane's entry
    float common = 0.0f;  // softmax without renormalisation: sum_i g_i s_i
    float mx = -INFINITY, sum = 0.0f;
    if (p.softmax && !p.renorm) {
      for (int i = lane; i < p.E; i += 32) mx = fmaxf(mx, to_f32(row[i]));
      mx = warp_max(mx);
      if (mx > -INFINITY)
        for (int i = lane; i < p.E; i += 32) sum += expf(to_f32(row[i]) - mx);
      sum = warp_sum(sum);
      const float s = l != -INFINITY ? expf(l - mx) / sum : 0.0f;
      common = warp_sum(g * s);
      d = s * (g - common);
    } else {
      const float top = warp_max(l);
      float s;  // score (softmax: relative to the largest chosen)
      if (p.softmax)
        s = l != -INFINITY ? expf(l - top) : 0.0f;
      else
        s = valid ? 1.0f / (1.0f + expf(-l)) : 0.0f;
      const float rest = p.softmax ? 1.0f : 1.0f / (1.0f + expf(l));  // 1 - s, without cancelling
      if (p.renorm) {
        const float total = warp_sum(s);
        const float pj = total == 0.0f ? 0.0f : s / total;
        const float mean = warp_sum(g * pj);
        d = (g - mean) * pj * rest;
      } else {
        d = g * s * rest;
      }
    }
    if (p.softmax && !p.renorm) {
      for (int i = lane; i < p.E; i += 32) {
        const float s = mx > -INFINITY ? expf(to_f32(row[i]) - mx) / sum : 0.0f;
        out[i] = from_f32<Tin>(-s * common);
      }
    } else if (vec) {
      uint4* o = reinterpret_cast<uint4*>(out);
      for (int i = lane; i < p.E / kVec; i += 32) o[i] = make_uint4(0, 0, 0, 0);
    } else {
      for (int i = lane; i < p.E; i += 32) out[i] = from_f32<Tin>(0.0f);
    }
    __syncwarp();  // the chosen entries are stored after the fill
    if (valid) out[e] = from_f32<Tin>(d);
  }
}

int grid_for(int64_t T) { return int(std::min<int64_t>(ceil_div(T, kWarps), 148 * 64)); }

template <int PL, typename Tin>
int launch_balanced(BalanceParams p, cudaStream_t s) {
  const int held = p.EG % PL == 0 ? p.EG / PL : 0;  // lanes that hold a group
  p.in_lanes = p.G > 1 && held > 0 && (held & (held - 1)) == 0;
  p.lanes_per_group = 32;
  while (p.in_lanes ? p.lanes_per_group > held : p.G * p.lanes_per_group > 32)
    p.lanes_per_group /= 2;
  p.group_shift = 0;
  while ((1 << p.group_shift) < p.lanes_per_group) ++p.group_shift;
  p.vec = p.E % PL == 0 && (p.E * sizeof(Tin)) % 16 == 0 && aligned16(p.logits);
  p.vec_bias = p.E % PL == 0 && aligned16(p.bias);
  const size_t smem = p.G > 1 && !p.in_lanes ? size_t(kWarps) * (p.E + p.G) * sizeof(double) : 0;
  KSW_LAUNCH(balanced_topk_kernel<PL, Tin>, dim3(grid_for(p.T)), dim3(32 * kWarps), smem, s, p);
  return MOE_OK;
}

template <typename Tin>
int launch_balanced_e(const BalanceParams& p, cudaStream_t s) {
  const int per = (p.E + 31) / 32;
  if (per <= 1) return launch_balanced<1, Tin>(p, s);
  if (per <= 2) return launch_balanced<2, Tin>(p, s);
  if (per <= 4) return launch_balanced<4, Tin>(p, s);
  if (per <= 8) return launch_balanced<8, Tin>(p, s);
  if (per <= 16) return launch_balanced<16, Tin>(p, s);
  return launch_balanced<32, Tin>(p, s);
}

template <typename Tin>
int launch_grad(const BalanceGradParams& p, cudaStream_t s) {
  KSW_LAUNCH(balanced_topk_grad_kernel<Tin>, dim3(grid_for(p.T)), dim3(32 * kWarps), 0, s, p);
  return MOE_OK;
}

int check_routing(int64_t num_tokens, int num_experts, int top_k, int ids_dtype,
                  int scoring_func) {
  KSW_REQUIRE(num_tokens >= 0, MOE_ERR_INVALID_ARG, "balanced_topk: num_tokens < 0");
  KSW_REQUIRE(num_experts >= 1 && num_experts <= 1024, MOE_ERR_UNSUPPORTED,
              "balanced_topk: num_experts must be in [1, 1024]");
  KSW_REQUIRE(top_k >= 1 && top_k <= 32 && top_k <= num_experts, MOE_ERR_UNSUPPORTED,
              "balanced_topk: top_k must be in [1, min(32, num_experts)]");
  KSW_REQUIRE(ids_dtype == MOE_DTYPE_I32 || ids_dtype == MOE_DTYPE_I64, MOE_ERR_INVALID_ARG,
              "balanced_topk: ids dtype must be int32 or int64");
  KSW_REQUIRE(scoring_func == 0 || scoring_func == 1, MOE_ERR_INVALID_ARG,
              "balanced_topk: scoring_func must be 0 (softmax) or 1 (sigmoid)");
  return MOE_OK;
}

}  // namespace
}  // namespace ksw

extern "C" int moe_balanced_topk(const void* router_logits, int logits_dtype,
                                 const float* expert_bias, int64_t num_tokens, int num_experts,
                                 int top_k, int renormalize, int num_expert_group,
                                 int topk_group, int group_score, int scoring_func,
                                 float routed_scaling_factor, void* topk_weights,
                                 int weights_dtype, void* topk_ids, int ids_dtype,
                                 int32_t* expert_load, void* stream) {
  using namespace ksw;
  int st = check_routing(num_tokens, num_experts, top_k, ids_dtype, scoring_func);
  if (st != MOE_OK) return st;
  KSW_REQUIRE(num_expert_group >= 1 && num_expert_group <= 32 &&
                  num_experts % num_expert_group == 0,
              MOE_ERR_UNSUPPORTED,
              "balanced_topk: num_expert_group must be in [1, 32] and divide num_experts");
  KSW_REQUIRE(topk_group >= 1 && topk_group <= num_expert_group, MOE_ERR_INVALID_ARG,
              "balanced_topk: topk_group must be in [1, num_expert_group]");
  KSW_REQUIRE(top_k <= topk_group * (num_experts / num_expert_group), MOE_ERR_UNSUPPORTED,
              "balanced_topk: top_k must fit in the kept groups");
  KSW_REQUIRE(group_score == 0 || group_score == 1, MOE_ERR_INVALID_ARG,
              "balanced_topk: group_score must be 0 (maximum) or 1 (sum of the two largest)");
  KSW_REQUIRE(weights_dtype == MOE_DTYPE_F32 || weights_dtype == MOE_DTYPE_F16 ||
                  weights_dtype == MOE_DTYPE_BF16,
              MOE_ERR_INVALID_ARG, "balanced_topk: weights dtype must be f32/bf16/f16");
  KSW_REQUIRE(logits_dtype == MOE_DTYPE_F32 || logits_dtype == MOE_DTYPE_F16 ||
                  logits_dtype == MOE_DTYPE_BF16,
              MOE_ERR_INVALID_ARG, "balanced_topk: logits dtype must be f32/bf16/f16");
  if ((st = check_device(nullptr)) != MOE_OK) return st;
  if (num_tokens == 0) return MOE_OK;
  KSW_REQUIRE(router_logits && topk_weights && topk_ids, MOE_ERR_INVALID_ARG,
              "balanced_topk: null pointer");
  BalanceParams p = {};
  p.logits = router_logits;
  p.bias = expert_bias;
  p.T = num_tokens;
  p.E = num_experts;
  p.k = top_k;
  p.G = num_expert_group;
  p.EG = num_experts / num_expert_group;
  p.kept = topk_group;
  p.eg_magic = uint32_t(((1 << 22) + p.EG - 1) / p.EG);
  p.softmax = scoring_func == 0;
  p.top2 = group_score;
  p.renorm = renormalize;
  p.scale = routed_scaling_factor;
  p.weights = topk_weights;
  p.w_dtype = weights_dtype;
  p.ids = topk_ids;
  p.ids64 = ids_dtype == MOE_DTYPE_I64;
  p.load = expert_load;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (logits_dtype == MOE_DTYPE_F32) return launch_balanced_e<float>(p, s);
  if (logits_dtype == MOE_DTYPE_BF16) return launch_balanced_e<__nv_bfloat16>(p, s);
  return launch_balanced_e<__half>(p, s);
}

extern "C" int moe_balanced_topk_backward(const void* router_logits, int logits_dtype,
                                          const void* topk_ids, int ids_dtype,
                                          const float* grad_weights, int64_t num_tokens,
                                          int num_experts, int top_k, int renormalize,
                                          int scoring_func, float routed_scaling_factor,
                                          void* grad_logits, void* stream) {
  using namespace ksw;
  int st = check_routing(num_tokens, num_experts, top_k, ids_dtype, scoring_func);
  if (st != MOE_OK) return st;
  KSW_REQUIRE(logits_dtype == MOE_DTYPE_F32 || logits_dtype == MOE_DTYPE_F16 ||
                  logits_dtype == MOE_DTYPE_BF16,
              MOE_ERR_INVALID_ARG, "balanced_topk_backward: logits dtype must be f32/bf16/f16");
  KSW_REQUIRE(aligned16(grad_logits), MOE_ERR_INVALID_ARG,
              "balanced_topk_backward: grad_logits must be 16-byte aligned");
  if ((st = check_device(nullptr)) != MOE_OK) return st;
  if (num_tokens == 0) return MOE_OK;
  KSW_REQUIRE(router_logits && topk_ids && grad_weights && grad_logits, MOE_ERR_INVALID_ARG,
              "balanced_topk_backward: null pointer");
  BalanceGradParams p = {};
  p.logits = router_logits;
  p.ids = topk_ids;
  p.ids64 = ids_dtype == MOE_DTYPE_I64;
  p.grad_weights = grad_weights;
  p.T = num_tokens;
  p.E = num_experts;
  p.k = top_k;
  p.softmax = scoring_func == 0;
  p.renorm = renormalize;
  p.scale = routed_scaling_factor;
  p.grad_logits = grad_logits;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (logits_dtype == MOE_DTYPE_F32) return launch_grad<float>(p, s);
  if (logits_dtype == MOE_DTYPE_BF16) return launch_grad<__nv_bfloat16>(p, s);
  return launch_grad<__half>(p, s);
}
