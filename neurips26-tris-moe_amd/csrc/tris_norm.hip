// Root-mean-square norm with the residual's addition.
//
//   h = x + residual,  residual_out = round(h),  out = round(h * rsqrt(mean(h^2) + eps) * (weight + offset))
//
// Everything between the loads and the one rounding of each output is fp32; the sum of squares of a row is a fixed
// tree, so results do not depend on the launch.
#include "tris_dtype.h"

namespace tris {

struct RmsNormArgs {
  const void* x;
  const void* residual;
  const void* weight;
  void* out;
  void* residual_out;
  int64_t x_stride, residual_stride, out_stride, residual_out_stride, rows;
  int32_t x_type, residual_type, weight_type, out_type, width;
  float weight_offset, eps;
};

// One workgroup a row, the row's values read twice.
__global__ __launch_bounds__(256) void rms_norm_kernel(const RmsNormArgs a) {
  __shared__ float part[4];
  const int64_t row = blockIdx.x;
  const auto sum_at = [&](int i) {
    const float x = load1(a.x, row * a.x_stride + i, a.x_type);
    return a.residual ? x + load1(a.residual, row * a.residual_stride + i, a.residual_type) : x;
  };
  float sq = 0.0f;
  for (int i = threadIdx.x; i < a.width; i += blockDim.x) {
    const float h = sum_at(i);
    sq += h * h;
  }
  sq = wave_sum_f32(sq);
  if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = sq;
  __syncthreads();
  sq = ((part[0] + part[1]) + part[2]) + part[3];
  const float f = rsqrtf(sq / static_cast<float>(a.width) + a.eps);
  for (int i = threadIdx.x; i < a.width; i += blockDim.x) {
    const float h = sum_at(i);
    const float w = load1(a.weight, i, a.weight_type) + a.weight_offset;
    if (a.residual) store1(a.residual_out, row * a.residual_out_stride + i, h, a.residual_type);
    store1(a.out, row * a.out_stride + i, h * f * w, a.out_type);
  }
}

}  // namespace tris

using namespace tris;

extern "C" int tris_rms_norm(const void* x, int32_t x_type, int64_t x_stride, const void* residual,
                             int32_t residual_type, int64_t residual_stride, const void* weight, int32_t weight_type,
                             float weight_offset, float eps, int64_t rows, int32_t width, void* out, int32_t out_type,
                             int64_t out_stride, void* residual_out, int64_t residual_out_stride, void* stream) {
  const char* who = "tris_rms_norm";
  TRIS_REQUIRE(rows >= 0 && width >= 1 && width <= 32768, "%s: rows must not be negative, width 1 to 32768", who);
  TRIS_REQUIRE(rows <= 2147483647LL, "%s: too many rows", who);
  TRIS_REQUIRE(is_16bit(x_type) && is_16bit(out_type) && (is_16bit(weight_type) || weight_type == TRIS_DTYPE_F32),
               "%s: x and out must be fp16 or bf16, weight one of these or fp32", who);
  if (rows == 0) return TRIS_OK;
  TRIS_REQUIRE(x && weight && out, "%s: null pointer", who);
  TRIS_REQUIRE((residual != nullptr) == (residual_out != nullptr), "%s: residual and residual_out go together", who);
  TRIS_REQUIRE(!residual || is_16bit(residual_type), "%s: residual must be fp16 or bf16", who);
  const auto apart = [&](int64_t stride) { return rows == 1 || stride >= width; };
  TRIS_REQUIRE(apart(out_stride) && (!residual || apart(residual_out_stride)), "%s: output rows overlap", who);
  TRIS_REQUIRE(rows == 1 || (x_stride >= 0 && residual_stride >= 0), "%s: negative stride", who);
  RmsNormArgs a{x, residual, weight, out, residual_out, x_stride, residual_stride, out_stride, residual_out_stride,
                rows, x_type, residual_type, weight_type, out_type, width, weight_offset, eps};
  hipLaunchKernelGGL(rms_norm_kernel, dim3(static_cast<unsigned>(rows)), dim3(256), 0,
                     static_cast<hipStream_t>(stream), a);
  return check_launch(who);
}
