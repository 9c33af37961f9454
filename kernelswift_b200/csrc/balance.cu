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
// One warp per token, the row in registers (lane l holds experts l, l + 32,
// ...). Group values are reduced from shared memory by 32 / G lanes per group
// at once. What bounds it: instruction issue and latency, not its T*E*4
// bytes.
#include <atomic>
#include <type_traits>

#include "common.cuh"

namespace ksw {
namespace {

constexpr int kMaxWarps = 4;  // warps (tokens) per block

struct BalanceParams {
  const void* logits;
  const float* bias;  // may be null
  int64_t T;
  int E, k, G, EG, kept;
  uint32_t eg_magic;  // ceil(2^22 / EG): e / EG = (e * eg_magic) >> 22 for e < 1024, EG <= 1024
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

// Largest value of a 32-bit key over the warp, and the smallest index among
// the lanes that hold it.
__device__ __forceinline__ uint32_t redux_max(uint32_t v) {
  return __reduce_max_sync(0xffffffffu, v);
}
__device__ __forceinline__ uint32_t redux_min(uint32_t v) {
  return __reduce_min_sync(0xffffffffu, v);
}
// Order-preserving map of floats to unsigned integers; 0 is below all of them.
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t u = __float_as_uint(v);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

// The warp's best (value, index): larger value, then lower index; lanes
// with i == INT32_MAX have nothing to offer.
__device__ __forceinline__ void warp_best(float& v, int& i) {
  const uint32_t key = i == INT32_MAX ? 0u : order_key(v);
  const uint32_t best = redux_max(key);
  i = int(redux_min(key == best ? uint32_t(i) : uint32_t(INT32_MAX)));
  v = key_value(best);
}
__device__ __forceinline__ void warp_best(double& v, int& i) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const double ov = __shfl_xor_sync(0xffffffffu, v, o);
    const int oi = __shfl_xor_sync(0xffffffffu, i, o);
    const bool take = oi != INT32_MAX && (i == INT32_MAX || ov > v || (ov == v && oi < i));
    if (take) {
      v = ov;
      i = oi;
    }
  }
}

template <typename R>
__device__ __forceinline__ R real_exp(R x);
template <>
__device__ __forceinline__ float real_exp<float>(float x) {
  return expf(x);
}
template <>
__device__ __forceinline__ double real_exp<double>(double x) {
  return exp(x);
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

// Error bound of the difference of two 32-bit c (per unit of the row's
// largest score, and of |c|): expf is off by 2 ulp at most, the sigmoid's add
// and divide by half a one each, the softmax's sum of up to 1024 terms by
// 37 / 2 ulp in the worst case; the sum with the bias rounds once more.
constexpr float kTolScore = 4e-6f, kTolValue = 4e-7f;

// Selects the row's experts in the arithmetic of R. Lane s < k returns the
// s-th expert in `sel`. Returns (32 bits only) whether some comparison was
// too close to trust. `mx` is the row's largest logit; `scratch` holds E + G
// values of R for this warp (groups only).
template <typename R, int PL, typename Tin>
__device__ bool select_row(const BalanceParams& p, const Tin* row, const float (&l)[PL], float mx,
                           int lane, R* scratch, int& sel) {
  constexpr bool kSingle = std::is_same<R, float>::value;
  R c[PL];
  R sum = R(0);
  const R rmx = mx == -INFINITY ? R(0) : R(mx);
  if (p.softmax) {
#pragma unroll
    for (int j = 0; j < PL; ++j) {
      c[j] = real_exp(R(l[j]) - rmx);
      if (lane + 32 * j < p.E) sum += c[j];
    }
    sum = warp_sum(sum);
  }
  const bool empty = p.softmax && mx == -INFINITY;  // no expert has a score
#pragma unroll
  for (int j = 0; j < PL; ++j) {
    const int e = lane + 32 * j;
    const R s = p.softmax ? (empty ? R(0) : c[j] / sum) : R(1) / (R(1) + real_exp(-R(l[j])));
    R v = s + (p.bias != nullptr && e < p.E ? R(__ldg(p.bias + e)) : R(0));
    c[j] = v != v ? R(-INFINITY) : v;  // a NaN ranks last
  }
  float smax = 0.0f;  // the row's largest score, for the error bound
  if constexpr (kSingle)
    smax = p.softmax ? (empty ? 0.0f : 1.0f / sum) : 1.0f / (1.0f + expf(-mx));
  bool close = false;

  uint32_t kept = 0xffffffffu;
  if (p.G > 1) {
    // position e + group keeps lanes of different groups on different banks
    __syncwarp();
#pragma unroll
    for (int j = 0; j < PL; ++j) {
      const int e = lane + 32 * j;
      if (e < p.E) scratch[e + group_of(p, e)] = c[j];
    }
    __syncwarp();
    int per = 32;  // lanes per group: the largest power of two that fits
    while (per * p.G > 32) per >>= 1;
    const int g = lane / per, sub = lane % per;
    R a = R(-INFINITY), b = R(-INFINITY);  // the two largest, a >= b
    if (g < p.G) {
      const R* at = scratch + g * (p.EG + 1);
      for (int i = sub; i < p.EG; i += per) {
        const R v = at[i];
        b = v > a ? a : (v > b ? v : b);
        a = v > a ? v : a;
      }
    }
    for (int o = per >> 1; o > 0; o >>= 1) {
      const R oa = __shfl_xor_sync(0xffffffffu, a, o);
      const R ob = __shfl_xor_sync(0xffffffffu, b, o);
      const R lo = a > oa ? oa : a;
      const R hb = b > ob ? b : ob;
      a = a > oa ? a : oa;
      b = lo > hb ? lo : hb;
    }
    // every lane of the group has its two largest; a group of one has no second
    R value = p.top2 && p.EG > 1 ? a + b : a;
    if (value != value) value = R(-INFINITY);  // +inf and -inf in one group
    const bool mine = g < p.G && sub == 0;
    kept = 0;
    bool taken = false;
    R last = R(0);
    for (int s = 0; s < p.kept; ++s) {
      R v = value;
      int i = mine && !taken ? g : INT32_MAX;
      warp_best(v, i);
      kept |= 1u << i;
      if (mine && g == i) taken = true;
      last = v;
    }
    if constexpr (kSingle) {
      const float tol = 2.0f * (kTolScore * smax + kTolValue * fabsf(last));
      close = mine && !taken && value >= last - tol && last > -INFINITY;
    }
  }

  uint32_t open = 0;  // bit j: expert lane + 32 j may still be chosen
#pragma unroll
  for (int j = 0; j < PL; ++j) {
    const int e = lane + 32 * j;
    const uint32_t g = p.G > 1 ? group_of(p, e) : 0u;
    if (e < p.E && ((kept >> g) & 1u)) open |= 1u << j;
  }
  sel = 0;
  R last = R(0);
  float last_l = 0.0f, last_b = 0.0f;
  for (int s = 0; s < p.k; ++s) {
    R v = R(-INFINITY);
    int i = INT32_MAX;
#pragma unroll
    for (int j = 0; j < PL; ++j)
      if (((open >> j) & 1u) && (i == INT32_MAX || c[j] > v)) {
        v = c[j];
        i = lane + 32 * j;
      }
    warp_best(v, i);
    if ((i & 31) == lane) open &= ~(1u << (i >> 5));
    if (lane == s) sel = i;
    if constexpr (kSingle) {
      // the pick's logit and bias: uniform loads of what the warp has read
      const float li = to_f32(row[i]);
      const float bi = p.bias != nullptr ? __ldg(p.bias + i) : 0.0f;
      if (s > 0 && last - v <= kTolScore * smax + kTolValue * fabsf(last) &&
          !(li == last_l && bi == last_b))
        close = true;
      last_l = li;
      last_b = bi;
    }
    last = v;
  }
  if constexpr (kSingle) {
    // the experts left out must be clear of the last one chosen
    const float bar = last - (kTolScore * smax + kTolValue * fabsf(last));
#pragma unroll
    for (int j = 0; j < PL; ++j) {
      const int e = lane + 32 * j;
      if (((open >> j) & 1u) && c[j] >= bar && last > -INFINITY &&
          !(l[j] == last_l && (p.bias == nullptr || __ldg(p.bias + e) == last_b)))
        close = true;
    }
    return __any_sync(0xffffffffu, close);
  }
  return false;
}

template <int PL, typename Tin>
__global__ void __launch_bounds__(32 * kMaxWarps)
    balanced_topk_kernel(const BalanceParams p) {
  extern __shared__ double s_scratch[];
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int warps = blockDim.x >> 5;
  double* scratch = s_scratch + (p.G > 1 ? warp * (p.E + p.G) : 0);
  for (int64_t t = int64_t(blockIdx.x) * warps + warp; t < p.T; t += int64_t(gridDim.x) * warps) {
    const Tin* row = static_cast<const Tin*>(p.logits) + t * p.E;
    float l[PL];
    float mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < PL; ++j) {
      const int e = lane + 32 * j;
      l[j] = e < p.E ? to_f32(row[e]) : -INFINITY;
      mx = fmaxf(mx, l[j]);
    }
    mx = warp_max(mx);
    int sel;
    if (select_row<float, PL>(p, row, l, mx, lane, reinterpret_cast<float*>(scratch), sel))
      select_row<double, PL>(p, row, l, mx, lane, scratch, sel);

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
// entry. Bound by the T*E*b bytes it writes (and reads, for the last form).
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
__global__ void __launch_bounds__(32 * kMaxWarps)
    balanced_topk_grad_kernel(const BalanceGradParams p) {
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int warps = blockDim.x >> 5;
  constexpr int kVec = 16 / int(sizeof(Tin));
  const bool vec = p.E % kVec == 0;  // every row starts on a 16-byte boundary
  for (int64_t t = int64_t(blockIdx.x) * warps + warp; t < p.T; t += int64_t(gridDim.x) * warps) {
    const Tin* row = static_cast<const Tin*>(p.logits) + t * p.E;
    Tin* out = static_cast<Tin*>(p.grad_logits) + t * p.E;
    const bool mine = lane < p.k;
    const int64_t at = t * p.k + lane;
    int e = 0;
    if (mine)
      e = p.ids64 ? int(static_cast<const int64_t*>(p.ids)[at])
                  : static_cast<const int32_t*>(p.ids)[at];
    const bool valid = mine && e >= 0 && e < p.E;  // an id out of range has no gradient
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

// One token per block while that leaves SMs free, else kMaxWarps tokens.
int pick_warps(int64_t T) { return T <= 148 * kMaxWarps ? 1 : kMaxWarps; }
int pick_grid(int64_t T, int warps) {
  return int(std::min<int64_t>(ceil_div(T, warps), 148 * 64));
}

template <int PL, typename Tin>
int launch_balanced(const BalanceParams& p, cudaStream_t s) {
  const int warps = pick_warps(p.T);
  const size_t smem = p.G > 1 ? size_t(warps) * (p.E + p.G) * sizeof(double) : 0;
  KSW_LAUNCH(balanced_topk_kernel<PL, Tin>, dim3(pick_grid(p.T, warps)), dim3(32 * warps), smem, s,
             p);
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
  const int warps = pick_warps(p.T);
  KSW_LAUNCH(balanced_topk_grad_kernel<Tin>, dim3(pick_grid(p.T, warps)), dim3(32 * warps), 0, s,
             p);
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
