// Quantisers of the dense block-scaled fp8 product (fp8_matmul.cu).
//
// Rows: each group of 128 columns of a row has one scale,
//   fp32:   s = absmax / 448 (1 for an all-zero group), q = e4m3 nearest to
//           x * 448 / absmax,
//   UE8M0:  s = 2^(b - 127), the least power of two with absmax / s <= 448
//           (b = 127 for an all-zero group), q = e4m3 nearest to x / s.
// With `gated` the row is silu(gate) * up of an input row [gate | up], so the
// down product's operand is written straight from the gate-up product.
// Blocks: the same with one scale for each 128 x 128 block (weights).
//
// x * 448 / absmax is the IEEE quotient (x * 0.875) / (absmax * 2^-9): for
// 16-bit inputs numerator and denominator are exact, so a quotient on the
// midpoint of two e4m3 values is recognised as such (a multiplication by a
// rounded reciprocal falls to either side of it).
//
// What bounds the row kernel: HBM (one B200: 4096 x 7168 bf16 14.4 us UE8M0, 6.1
// TB/s, and 17.1 us fp32 scales; 8192 x 8192 f32 47.8 us, 7.0 TB/s), for the gated
// form instruction issue too (4096 x 2048 11.5 us, 3.6 TB/s); a few rows are
// latency (1 x 7168 1.2 us). A half-warp holds a group (8 columns per
// lane, one 16-byte load for 16-bit inputs, two where rows start off such a
// boundary), a warp up to 1024 columns of a row with its loads in flight before
// the first is used; neighbouring warps take neighbouring columns, so that a
// block reads one run of memory.
#include <type_traits>

#include "common.cuh"

namespace ksw {
namespace {

constexpr int kRowWarps = 8;

struct QuantRows {
  const void* x;
  int64_t T, K, ld_x;
  uint8_t* q;
  int64_t ld_q;
  void* scale;
  int64_t s_row, s_blk;  // strides of the scale, in elements
};

// Eight consecutive elements, as the aligned 16-byte vectors that hold them
// (each holds at least one of their bytes) and, unless all rows start on such
// boundaries (ALIGNED), the offset of the first byte, which the lanes of a row
// share.
template <typename Tin, bool ALIGNED>
struct Raw8 {
  static constexpr int kVecs = int(sizeof(Tin)) / 2 + (ALIGNED ? 0 : 1);
  uint4 w[kVecs];

  __device__ __forceinline__ void load(const Tin* p) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    const uint4* base = reinterpret_cast<const uint4*>(at & ~uintptr_t(15));
#pragma unroll
    for (int i = 0; i < int(sizeof(Tin)) / 2; ++i) w[i] = __ldg(base + i);
    if constexpr (!ALIGNED)
      w[kVecs - 1] = (at & 15) ? __ldg(base + kVecs - 1) : make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void values(uint32_t offset, float (&v)[8]) const {
    constexpr int kIn = 4 * kVecs, kOut = 2 * int(sizeof(Tin));
    uint32_t x[kIn];
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      x[4 * i] = w[i].x, x[4 * i + 1] = w[i].y, x[4 * i + 2] = w[i].z, x[4 * i + 3] = w[i].w;
    }
    if constexpr (!ALIGNED) {
      // a shift by whole words, then by the bytes that are left
      if (offset & 8) {
#pragma unroll
        for (int i = 0; i + 2 < kIn; ++i) x[i] = x[i + 2];
      }
      if (offset & 4) {
#pragma unroll
        for (int i = 0; i + 1 < kIn; ++i) x[i] = x[i + 1];
      }
      if constexpr (sizeof(Tin) == 2) {
#pragma unroll
        for (int i = 0; i < kOut; ++i) x[i] = __funnelshift_r(x[i], x[i + 1], 8 * (offset & 3));
      }
    }
    const Tin* e = reinterpret_cast<const Tin*>(x);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32(e[i]);
  }
};
// Eight consecutive elements, one by one, of which `n` exist (the rest are 0).
template <typename Tin>
__device__ __forceinline__ void load8(const Tin* p, int64_t n, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = i < n ? to_f32(p[i]) : 0.0f;
}

// 1 / x to an ulp, for a normal result.
__device__ __forceinline__ float rcp_ulp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two fp32 operations per instruction, each rounded as by itself.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// silu(g) * u with sigmoid(g) = 1 / (1 + e^-g), for negative g e^g / (1 + e^g):
// the exponential never overflows and the divisor lies between 1 and 2, where
// the fast reciprocal is off by an ulp. exp 2 ulp, its sum and the products half
// an ulp each: under 6 in all, from a gate of -87 on (e^g is subnormal below).
__device__ __forceinline__ float2 silu_up(float2 g, float2 u) {
  const float2 e = make_float2(expf(-fabsf(g.x)), expf(-fabsf(g.y)));
  const float2 r = make_float2(rcp_ulp(1.0f + e.x), rcp_ulp(1.0f + e.y));
  const float2 n = mul2(e, r);
  const float2 s = make_float2(g.x < 0.0f ? n.x : r.x, g.y < 0.0f ? n.y : r.y);
  return mul2(mul2(g, s), u);
}
__device__ __forceinline__ double silu_up(double g, double u) { return g / (1.0 + exp(-g)) * u; }

// Largest of eight gated values in 64 bits, `n` of which exist. Out of line: few
// warps come here, and its registers would cost all of them their number.
template <typename Tin>
__device__ __noinline__ double gated_top(const Tin* g, const Tin* u, int64_t n) {
  double top = 0.0;
#pragma unroll 1
  for (int e = 0; e < 8 && e < n; ++e)
    top = fmax(top, fabs(silu_up(double(to_f32(g[e])), double(to_f32(u[e])))));
  return top;
}

// Two e4m3 bytes, round to nearest even; a NaN stays one, beyond 448 saturates.
__device__ __forceinline__ uint32_t e4m3x2(float a, float b) {
  return uint32_t(__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3));
}

// The factors of x * 448 / amax = (x * num) / den; up keeps den, and residuals
// of quotients down to e4m3's least, out of the subnormal range.
struct Ratio {
  float num, den;
};
__device__ __forceinline__ Ratio ratio_of(float amax) {
  if (!(amax > 0.0f)) return {0.875f, 0.875f};
  const float up = amax < 0x1p-60f ? 0x1p100f : 1.0f;
  return {0.875f * up, amax * up * 0x1p-9f};
}
// a / den: q = a y is off by two ulp at most for a y = 1 / den within an ulp; the
// residual a - q den is exact in one fma (but for its last bit), and q + residual
// * y rounds to the quotient, with an error of 2^-21 ulp before that rounding. A
// quotient on the midpoint of two e4m3 values, which 32 bits hold, so comes out
// on it. minus is -den, or 0 for an infinite den, whose finite quotients are q = 0.
__device__ __forceinline__ float2 quotient(float2 a, float minus, float y) {
  const float2 q = mul2(a, both(y));
  return fma2(fma2(q, both(minus), a), both(y), q);
}
__device__ __forceinline__ float fp32_scale(float amax) {
  if (amax >= 0x1p-100f && amax < INFINITY) return quotient(both(amax), -448.0f, 1.0f / 448.0f).x;
  return amax > 0.0f ? amax / 448.0f : 1.0f;
}

// Maxima of ITERS groups over the 16 lanes of each half-warp; lane l of a half
// gets that of group l / (16 / ITERS). While lanes hold several groups, each
// step hands half of them to the lane that keeps those.
template <int ITERS>
__device__ __forceinline__ float group_max(float (&m)[ITERS], int lane) {
  if constexpr (ITERS == 4) {
    const bool up = lane & 8;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float got = __shfl_xor_sync(0xffffffffu, up ? m[i] : m[i + 2], 8);
      m[i] = fmaxf(up ? m[i + 2] : m[i], got);
    }
  }
  if constexpr (ITERS >= 2) {
    constexpr int o = ITERS == 4 ? 4 : 8;
    const bool up = lane & o;
    const float got = __shfl_xor_sync(0xffffffffu, up ? m[0] : m[1], o);
    m[0] = fmaxf(up ? m[1] : m[0], got);
  }
#pragma unroll
  for (int o = 8 / ITERS; o > 0; o >>= 1)
    m[0] = fmaxf(m[0], __shfl_xor_sync(0xffffffffu, m[0], o));
  return m[0];
}

// ITERS: runs of 256 columns per warp. One row's warps follow one another.
template <typename Tin, bool ALIGNED, bool GATED, bool UE8M0, int ITERS>
__global__ void __launch_bounds__(32 * kRowWarps)
    fp8_quantize_rows_kernel(const QuantRows p, uint32_t chunks) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const uint32_t unit = blockIdx.x * kRowWarps + (threadIdx.x >> 5);
  const int64_t t = unit / chunks;
  if (t >= p.T) return;
  const int64_t c0 = int64_t(unit - uint32_t(t) * chunks) * (256 * ITERS) + 8 * lane;
  const Tin* row = static_cast<const Tin*>(p.x) + t * p.ld_x;
  float v[ITERS][8];
  float u[GATED ? ITERS : 1][8];
  const uint32_t off = uint32_t(reinterpret_cast<uintptr_t>(row)) & 15u;
  const uint32_t off_u = uint32_t(reinterpret_cast<uintptr_t>(row + p.K)) & 15u;
  Raw8<Tin, ALIGNED> raw[ITERS], raw_u[GATED ? ITERS : 1];
  // one branch for the warp, not one per load: the loads go out together
  const bool whole = c0 - 8 * lane + 256 * ITERS <= p.K;
  if (whole) {
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
      raw[i].load(row + c0 + 256 * i);
      if constexpr (GATED) raw_u[i].load(row + p.K + c0 + 256 * i);
    }
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
      raw[i].values(off, v[i]);
      if constexpr (GATED) raw_u[i].values(off_u, u[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
      const int64_t c = c0 + 256 * i;
      if (c + 8 <= p.K) {
        raw[0].load(row + c);
        raw[0].values(off, v[i]);
        if constexpr (GATED) {
          raw_u[0].load(row + p.K + c);
          raw_u[0].values(off_u, u[i]);
        }
      } else {
        load8(row + c, p.K - c, v[i]);
        if constexpr (GATED) load8(row + p.K + c, p.K - c, u[i]);
      }
    }
  }
  float m[ITERS];
#pragma unroll
  for (int i = 0; i < ITERS; ++i) {
    m[i] = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      if constexpr (GATED) {
        const float2 s = silu_up(make_float2(v[i][e], v[i][e + 1]),
                                 make_float2(u[i][e], u[i][e + 1]));
        v[i][e] = s.x;
        v[i][e + 1] = s.y;
      }
      m[i] = fmaxf(m[i], fmaxf(fabsf(v[i][e]), fabsf(v[i][e + 1])));
    }
  }
  // From here to the factors of the elements a lane works on one group of its
  // half-warp, that of run i = my_run.
  constexpr int kShare = 16 / ITERS;  // lanes per group
  const float amax = group_max<ITERS>(m, lane);
  const int my_run = (lane & 15) / kShare;
  const int64_t col = c0 - 8 * (lane & 15) + 256 * my_run;
  const bool writer = (lane & (kShare - 1)) == 0 && col < p.K;
  const int64_t at = t * p.s_row + col / 128 * p.s_blk;
  float f0, f1 = 0.0f, f2 = 0.0f;
  if constexpr (UE8M0) {
    uint32_t b = ue8m0_byte(amax);
    if constexpr (GATED) {
      // a maximum within the rounding of the 32-bit silu (under 8 ulp) of
      // 448 * 2^k decides the scale by its 64-bit value
      const uint32_t bits = __float_as_uint(amax);
      const int ulps = int(bits & 0x7fffffu) - 0x600000;
      const bool near = amax > 0.0f && amax < INFINITY && ulps >= -16 && ulps <= 16;
      if (__any_sync(0xffffffffu, near)) {
#pragma unroll 1
        for (int i = 0; i < ITERS; ++i) {
          const int64_t c = c0 + 256 * i;
          double top = gated_top(row + c, row + p.K + c, p.K - c);
#pragma unroll
          for (int o = 8; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
          if (near && i == my_run) {
            const int e = int(bits >> 23);
            b = uint32_t(min(max(e - 8 + (top > ldexp(1.75, e - 127) ? 1 : 0), 0), 254));
          }
        }
      }
    }
    f0 = ue8m0_inv_scale(b);
    if (writer) static_cast<uint8_t*>(p.scale)[at] = uint8_t(b);
  } else {
    const Ratio r = ratio_of(amax);
    f0 = r.num;
    f1 = amax < INFINITY ? -r.den : 0.0f;
    f2 = rcp_ulp(r.den);
    if (writer) static_cast<float*>(p.scale)[at] = fp32_scale(amax);
  }
#pragma unroll
  for (int i = 0; i < ITERS; ++i) {
    const int src = (lane & 16) + kShare * i;
    const float x0 = __shfl_sync(0xffffffffu, f0, src);
    const float x1 = UE8M0 ? 0.0f : __shfl_sync(0xffffffffu, f1, src);
    const float x2 = UE8M0 ? 0.0f : __shfl_sync(0xffffffffu, f2, src);
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float2 a = mul2(make_float2(v[i][2 * e], v[i][2 * e + 1]), both(x0));
      if constexpr (!UE8M0) a = quotient(a, x1, x2);
      w[e] = e4m3x2(a.x, a.y);
    }
    // rows of q start on 16-byte boundaries and are padded to 16 bytes, so
    // 8 bytes at a column below K are inside the row
    if (c0 + 256 * i < p.K)
      *reinterpret_cast<uint2*>(p.q + t * p.ld_q + c0 + 256 * i) =
          make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
  }
}

// One block per 128 x 128 block of the matrix: 8 warps of 16 rows, lane l
// holds columns l, l + 32, ... of each row. One-time work (weights), in loads of one
// element and stores of one byte per lane: 4096 x 7168 bf16 38 us in UE8M0 (2.3
// TB/s), 58 us with fp32 scales (a division per element); f32 35 and 54 us.
constexpr int kBlkWarps = 8;

template <typename Tin, bool UE8M0>
__global__ void __launch_bounds__(32 * kBlkWarps)
    fp8_quantize_blocks_kernel(const Tin* __restrict__ w, int64_t N, int64_t K, int64_t ld_w,
                               uint8_t* __restrict__ q, int64_t ld_q, void* scale,
                               int64_t col_blocks) {
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t nb = blockIdx.x / col_blocks, kb = blockIdx.x % col_blocks;
  __shared__ float s_max[kBlkWarps];
  float v[16][4];
  float amax = 0.0f;
#pragma unroll
  for (int r = 0; r < 16; ++r)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t n = nb * 128 + warp * 16 + r, k = kb * 128 + lane + 32 * j;
      v[r][j] = n < N && k < K ? to_f32(w[n * ld_w + k]) : 0.0f;
      amax = fmaxf(amax, fabsf(v[r][j]));
    }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if (lane == 0) s_max[warp] = amax;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kBlkWarps; ++i) amax = fmaxf(amax, s_max[i]);
  Ratio ratio = ratio_of(amax);
  if constexpr (UE8M0) {
    const uint32_t b = ue8m0_byte(amax);
    ratio = {ue8m0_inv_scale(b), 1.0f};
    if (threadIdx.x == 0) static_cast<uint8_t*>(scale)[blockIdx.x] = uint8_t(b);
  } else {
    if (threadIdx.x == 0) static_cast<float*>(scale)[blockIdx.x] = fp32_scale(amax);
  }
#pragma unroll
  for (int r = 0; r < 16; ++r)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t n = nb * 128 + warp * 16 + r, k = kb * 128 + lane + 32 * j;
      const float x = v[r][j] * ratio.num;
      if (n < N && k < K)
        q[n * ld_q + k] = uint8_t(e4m3x2(UE8M0 ? x : x / ratio.den, 0.0f));
    }
}

template <typename Tin, bool ALIGNED, bool GATED, int ITERS>
int launch_rows_i(const QuantRows& p, int ue8m0, cudaStream_t s) {
  const int64_t chunks = ceil_div(p.K, 256 * ITERS);
  const int64_t blocks = ceil_div(p.T * chunks, kRowWarps);
  KSW_REQUIRE(blocks * kRowWarps < (int64_t(1) << 32), MOE_ERR_UNSUPPORTED,
              "fp8_quantize_rows: too many elements");
  if (ue8m0)
    KSW_LAUNCH(fp8_quantize_rows_kernel<Tin, ALIGNED, GATED, true, ITERS>, dim3(unsigned(blocks)),
               dim3(32 * kRowWarps), 0, s, p, uint32_t(chunks));
  else
    KSW_LAUNCH(fp8_quantize_rows_kernel<Tin, ALIGNED, GATED, false, ITERS>, dim3(unsigned(blocks)),
               dim3(32 * kRowWarps), 0, s, p, uint32_t(chunks));
  return MOE_OK;
}

template <typename Tin, bool ALIGNED, bool GATED>
int launch_rows(const QuantRows& p, int ue8m0, cudaStream_t s) {
  // 256 columns per warp until the SMs are full of warps, then more loads in
  // flight per warp and, for 16-bit inputs, maxima of four groups reduced
  // together. One B200, bf16 x 7168 columns, UE8M0: 64 rows 1.8 us against 1.9
  // with 1024 columns per warp, 600 rows 4.2 against 3.8, 4096 rows 20.4 against
  // 14.4; f32 8192 x 8192 49.8 us with 256, 47.8 with 512, 47.9 with 1024; gated
  // 4096 x 2048 13.5, 11.5, 12.7.
  constexpr int kMany = GATED || sizeof(Tin) == 4 ? 2 : 4;
  if (p.T * ceil_div(p.K, 256) <= 148 * 64)
    return launch_rows_i<Tin, ALIGNED, GATED, 1>(p, ue8m0, s);
  return launch_rows_i<Tin, ALIGNED, GATED, kMany>(p, ue8m0, s);
}

template <typename Tin>
int launch_rows_t(const QuantRows& p, int gated, int ue8m0, cudaStream_t s) {
  const bool aligned = aligned16(p.x) && (p.ld_x * sizeof(Tin)) % 16 == 0 &&
                       (!gated || (p.K * sizeof(Tin)) % 16 == 0);
  if (gated)
    return aligned ? launch_rows<Tin, true, true>(p, ue8m0, s)
                   : launch_rows<Tin, false, true>(p, ue8m0, s);
  return aligned ? launch_rows<Tin, true, false>(p, ue8m0, s)
                 : launch_rows<Tin, false, false>(p, ue8m0, s);
}

template <typename Tin>
int launch_blocks(const void* w, int64_t N, int64_t K, int64_t ld_w, int ue8m0, uint8_t* q,
                  int64_t ld_q, void* scale, cudaStream_t s) {
  const int64_t kb = ceil_div(K, 128), blocks = ceil_div(N, 128) * kb;
  if (ue8m0)
    KSW_LAUNCH(fp8_quantize_blocks_kernel<Tin, true>, dim3(unsigned(blocks)),
               dim3(32 * kBlkWarps), 0, s, static_cast<const Tin*>(w), N, K, ld_w, q, ld_q, scale,
               kb);
  else
    KSW_LAUNCH(fp8_quantize_blocks_kernel<Tin, false>, dim3(unsigned(blocks)),
               dim3(32 * kBlkWarps), 0, s, static_cast<const Tin*>(w), N, K, ld_w, q, ld_q, scale,
               kb);
  return MOE_OK;
}

int check_source(const char* what, int dtype, int64_t rows, int64_t cols, int64_t ld,
                 int64_t wide, int scale_format, const void* q, int64_t ld_q) {
  const std::string name(what);
  KSW_REQUIRE(dtype == MOE_DTYPE_F32 || dtype == MOE_DTYPE_F16 || dtype == MOE_DTYPE_BF16,
              MOE_ERR_INVALID_ARG, name + ": source dtype must be f32/f16/bf16");
  KSW_REQUIRE(rows >= 0 && cols >= 1, MOE_ERR_INVALID_ARG, name + ": bad sizes");
  KSW_REQUIRE(rows <= (int64_t(1) << 31) - 8 && cols <= (int64_t(1) << 31) - 8,
              MOE_ERR_UNSUPPORTED, name + ": sizes beyond 2^31");
  KSW_REQUIRE(ld >= wide, MOE_ERR_INVALID_ARG, name + ": row stride shorter than a row");
  KSW_REQUIRE(scale_format == 0 || scale_format == 1, MOE_ERR_INVALID_ARG,
              name + ": scale_format must be 0 (fp32) or 1 (UE8M0)");
  KSW_REQUIRE(aligned16(q) && ld_q % 16 == 0 && ld_q >= round_up(cols, 16), MOE_ERR_INVALID_ARG,
              name + ": the fp8 rows must start on 16-byte boundaries");
  return MOE_OK;
}

}  // namespace
}  // namespace ksw

extern "C" int moe_fp8_quantize_rows(const void* x, int x_dtype, int64_t num_rows, int64_t cols,
                                     int64_t ld_x, int gated, int scale_format, void* q,
                                     int64_t ld_q, void* scale, int64_t scale_row_stride,
                                     int64_t scale_block_stride, void* stream) {
  using namespace ksw;
  int st = check_source("fp8_quantize_rows", x_dtype, num_rows, cols, ld_x,
                        gated ? 2 * cols : cols, scale_format, q, ld_q);
  if (st != MOE_OK) return st;
  if ((st = check_device(nullptr)) != MOE_OK) return st;
  if (num_rows == 0) return MOE_OK;
  KSW_REQUIRE(x && q && scale, MOE_ERR_INVALID_ARG, "fp8_quantize_rows: null pointer");
  const QuantRows p = {x,    num_rows,         cols, ld_x, static_cast<uint8_t*>(q), ld_q, scale,
                       scale_row_stride, scale_block_stride};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (x_dtype == MOE_DTYPE_F32) return launch_rows_t<float>(p, gated, scale_format, s);
  if (x_dtype == MOE_DTYPE_BF16) return launch_rows_t<__nv_bfloat16>(p, gated, scale_format, s);
  return launch_rows_t<__half>(p, gated, scale_format, s);
}

extern "C" int moe_fp8_quantize_blocks(const void* w, int w_dtype, int64_t rows, int64_t cols,
                                       int64_t ld_w, int scale_format, void* q, int64_t ld_q,
                                       void* scale, void* stream) {
  using namespace ksw;
  int st = check_source("fp8_quantize_blocks", w_dtype, rows, cols, ld_w, cols, scale_format, q,
                        ld_q);
  if (st != MOE_OK) return st;
  KSW_REQUIRE(ceil_div(rows, 128) * ceil_div(cols, 128) < (int64_t(1) << 31),
              MOE_ERR_UNSUPPORTED, "fp8_quantize_blocks: too many blocks");
  if ((st = check_device(nullptr)) != MOE_OK) return st;
  if (rows == 0) return MOE_OK;
  KSW_REQUIRE(w && q && scale, MOE_ERR_INVALID_ARG, "fp8_quantize_blocks: null pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  uint8_t* qb = static_cast<uint8_t*>(q);
  if (w_dtype == MOE_DTYPE_F32)
    return launch_blocks<float>(w, rows, cols, ld_w, scale_format, qb, ld_q, scale, s);
  if (w_dtype == MOE_DTYPE_BF16)
    return launch_blocks<__nv_bfloat16>(w, rows, cols, ld_w, scale_format, qb, ld_q, scale, s);
  return launch_blocks<__half>(w, rows, cols, ld_w, scale_format, qb, ld_q, scale, s);
}
