// The SwiGLU MLP of a shared expert on block-scaled fp8 weights: four launches
// on one workspace (quantise, gate-up product, silu(gate) * up quantised, down
// product with the addend in its epilogue). What bounds it: at a few tokens
// the stream of 3 H I weight bytes plus the launches, at many tokens the two
// products. One B200, 7168 x 2048, back to back, UE8M0 and fp32 scales: 1 token 21.0
// and 21.3 us, 16 tokens 21.8 and 22.5 us (44 MB of weights), 64 tokens 24.2 and 26.5
// us, 2048 tokens 87 us (2070 TFLOP/s) and 114 us; with an addend 16 tokens take 22.2
// and 22.9 us, 2048 tokens 92 and 127 us.
#include "common.cuh"

namespace ksw {
namespace {

// Pieces of the workspace, each on a 256-byte boundary.
struct MlpLayout {
  int64_t ld_x, ld_act;    // pitches of the quantised rows
  int64_t xs_row, xs_blk;  // scale strides: by block for fp32, by row for UE8M0
  int64_t as_row, as_blk;
  size_t x, xs, both, act, as, bytes;
};

MlpLayout mlp_layout(int64_t T, int64_t H, int64_t I, int dtype, int scale_format) {
  MlpLayout l = {};
  const int64_t elem = dtype == MOE_DTYPE_F32 ? 4 : 2;
  const int64_t xb = ceil_div(H, 128), ab = ceil_div(I, 128);
  l.ld_x = round_up(H, 16);
  l.ld_act = round_up(I, 16);
  size_t at = 0;
  auto take = [&](int64_t bytes) {
    const size_t here = at;
    at += align256(size_t(bytes));
    return here;
  };
  l.x = take(T * l.ld_x);
  if (scale_format == 0) {
    l.xs_row = l.as_row = 1;
    l.xs_blk = l.as_blk = round_up(T, 4);
    l.xs = take(xb * l.xs_blk * 4);
    l.as = take(ab * l.as_blk * 4);
  } else {
    l.xs_row = round_up(xb, 4);
    l.as_row = round_up(ab, 4);
    l.xs_blk = l.as_blk = 1;
    l.xs = take(T * l.xs_row);
    l.as = take(T * l.as_row);
  }
  l.both = take(T * 2 * I * elem);
  l.act = take(T * l.ld_act);
  l.bytes = at;
  return l;
}

int check_mlp(int64_t T, int64_t H, int64_t I, int dtype, int scale_format) {
  KSW_REQUIRE(T >= 0 && H >= 1 && I >= 1, MOE_ERR_INVALID_ARG, "fp8_swiglu_mlp: bad sizes");
  KSW_REQUIRE(T < (int64_t(1) << 30) && H < (int64_t(1) << 30) && I < (int64_t(1) << 29),
              MOE_ERR_UNSUPPORTED, "fp8_swiglu_mlp: sizes beyond 2^30");
  KSW_REQUIRE(dtype == MOE_DTYPE_F32 || dtype == MOE_DTYPE_F16 || dtype == MOE_DTYPE_BF16,
              MOE_ERR_INVALID_ARG, "fp8_swiglu_mlp: dtype must be f32/f16/bf16");
  KSW_REQUIRE(scale_format == 0 || scale_format == 1, MOE_ERR_INVALID_ARG,
              "fp8_swiglu_mlp: scale_format must be 0 (fp32) or 1 (UE8M0)");
  return MOE_OK;
}

}  // namespace
}  // namespace ksw

extern "C" int moe_fp8_swiglu_mlp_workspace_size(int64_t num_rows, int64_t hidden, int64_t inter,
                                                 int dtype, int scale_format, size_t* bytes) {
  using namespace ksw;
  int st = check_mlp(num_rows, hidden, inter, dtype, scale_format);
  if (st != MOE_OK) return st;
  KSW_REQUIRE(bytes != nullptr, MOE_ERR_INVALID_ARG, "fp8_swiglu_mlp: null pointer");
  *bytes = mlp_layout(num_rows, hidden, inter, dtype, scale_format).bytes;
  return MOE_OK;
}

extern "C" int moe_fp8_swiglu_mlp(const void* x, int64_t ld_x, int dtype, int64_t num_rows,
                                  int64_t hidden, int64_t inter, const void* w13, int64_t ld_w13,
                                  const void* w13_scale, const void* w2, int64_t ld_w2,
                                  const void* w2_scale, int scale_format, const void* addend,
                                  int64_t ld_addend, void* out, int64_t ld_out, void* workspace,
                                  size_t workspace_bytes, int32_t* status, void* stream) {
  using namespace ksw;
  int st = check_mlp(num_rows, hidden, inter, dtype, scale_format);
  if (st != MOE_OK) return st;
  const MlpLayout l = mlp_layout(num_rows, hidden, inter, dtype, scale_format);
  KSW_REQUIRE(ld_x >= hidden && ld_out >= hidden && (addend == nullptr || ld_addend >= hidden) &&
                  ld_w13 >= hidden && ld_w2 >= inter,
              MOE_ERR_INVALID_ARG, "fp8_swiglu_mlp: row stride shorter than a row");
  KSW_REQUIRE(ld_w13 % 16 == 0 && ld_w2 % 16 == 0 && aligned16(w13) && aligned16(w2),
              MOE_ERR_INVALID_ARG,
              "fp8_swiglu_mlp: the fp8 rows must start on 16-byte boundaries");
  if (num_rows == 0) return check_device(nullptr);
  KSW_REQUIRE(x && w13 && w13_scale && w2 && w2_scale && out, MOE_ERR_INVALID_ARG,
              "fp8_swiglu_mlp: null pointer");
  KSW_REQUIRE(workspace != nullptr && workspace_bytes >= l.bytes, MOE_ERR_WORKSPACE,
              "fp8_swiglu_mlp: workspace missing or too small");
  KSW_REQUIRE(aligned16(workspace), MOE_ERR_INVALID_ARG,
              "fp8_swiglu_mlp: workspace must be 16-byte aligned");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  st = moe_fp8_quantize_rows(x, dtype, num_rows, hidden, ld_x, 0, scale_format, ws + l.x, l.ld_x,
                             ws + l.xs, l.xs_row, l.xs_blk, stream);
  if (st != MOE_OK) return st;
  st = moe_fp8_matmul(ws + l.x, l.ld_x, ws + l.xs, l.xs_row, l.xs_blk, w13, ld_w13, w13_scale,
                      scale_format, num_rows, 2 * inter, hidden, nullptr, 0, ws + l.both,
                      2 * inter, dtype, status, stream);
  if (st != MOE_OK) return st;
  st = moe_fp8_quantize_rows(ws + l.both, dtype, num_rows, inter, 2 * inter, 1, scale_format,
                             ws + l.act, l.ld_act, ws + l.as, l.as_row, l.as_blk, stream);
  if (st != MOE_OK) return st;
  return moe_fp8_matmul(ws + l.act, l.ld_act, ws + l.as, l.as_row, l.as_blk, w2, ld_w2, w2_scale,
                        scale_format, num_rows, hidden, inter, addend, ld_addend, out, ld_out,
                        dtype, status, stream);
}
