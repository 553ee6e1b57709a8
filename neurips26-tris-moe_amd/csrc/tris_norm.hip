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

// kLanes threads a row, each with kChunks runs of eight columns in registers, so that a row is read once.  Up to 64
// lanes a row a workgroup has 256 / kLanes rows and a row's sum stays in its wavefront; above, a row has the workgroup.
// kVector: every row is 16-byte aligned and the width a multiple of eight: 16-byte loads; else one value at a time, a
// thread's columns kLanes apart.
template <int kLanes, int kChunks, bool kVector>
__global__ __launch_bounds__(kLanes > 256 ? kLanes : 256) void rms_norm_kernel(const RmsNormArgs a) {
  constexpr int kRows = kLanes <= kWave ? 256 / kLanes : 1;
  const int t = threadIdx.x % kLanes;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / kLanes;
  const bool live = row < a.rows;
  const bool x_bf16 = a.x_type == TRIS_DTYPE_BF16, r_bf16 = a.residual_type == TRIS_DTYPE_BF16;
  const auto column = [&](int c, int e) { return kVector ? (c * kLanes + t) * 8 : (c * 8 + e) * kLanes + t; };
  float h[kChunks][8], w[kChunks][8];
  // the row and the weights in flight together
  uint4 xs[kChunks], rs[kChunks], ws[kChunks], ws2[kChunks];
  if constexpr (kVector) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int i = column(c, 0);
      if (!live || i >= a.width) continue;
      xs[c] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.x) + row * a.x_stride + i);
      if (a.residual)
        rs[c] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.residual) + row * a.residual_stride + i);
      if (a.weight_type == TRIS_DTYPE_F32) {
        ws[c] = *reinterpret_cast<const uint4*>(static_cast<const float*>(a.weight) + i);
        ws2[c] = *reinterpret_cast<const uint4*>(static_cast<const float*>(a.weight) + i + 4);
      } else {
        ws[c] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.weight) + i);
      }
    }
  }
  float sq = 0.0f;
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    if constexpr (kVector) {
      const int i = column(c, 0);
      if (!live || i >= a.width) continue;
      widen8(xs[c], x_bf16, h[c]);
      if (a.residual) {
        float r[8];
        widen8(rs[c], r_bf16, r);
#pragma unroll
        for (int e = 0; e < 8; ++e) h[c][e] += r[e];
      }
      if (a.weight_type == TRIS_DTYPE_F32) {
        const uint32_t u[8] = {ws[c].x, ws[c].y, ws[c].z, ws[c].w, ws2[c].x, ws2[c].y, ws2[c].z, ws2[c].w};
#pragma unroll
        for (int e = 0; e < 8; ++e) w[c][e] = __uint_as_float(u[e]);
      } else {
        widen8(ws[c], a.weight_type == TRIS_DTYPE_BF16, w[c]);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) sq += h[c][e] * h[c][e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int i = column(c, e);
        h[c][e] = w[c][e] = 0.0f;
        if (!live || i >= a.width) continue;
        h[c][e] = load1(a.x, row * a.x_stride + i, a.x_type);
        if (a.residual) h[c][e] += load1(a.residual, row * a.residual_stride + i, a.residual_type);
        w[c][e] = load1(a.weight, i, a.weight_type);
        sq += h[c][e] * h[c][e];
      }
    }
  }
  if constexpr (kLanes < kWave) {
#pragma unroll
    for (int d = 1; d < kLanes; d *= 2) sq += __shfl_xor(sq, d);
  } else {
    sq = wave_sum_f32(sq);
    if constexpr (kLanes > kWave) {
      __shared__ float part[kLanes / kWave];
      if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = sq;
      __syncthreads();
      sq = part[0];
#pragma unroll
      for (int i = 1; i < kLanes / kWave; ++i) sq += part[i];
    }
  }
  const float f = rsqrtf(sq / static_cast<float>(a.width) + a.eps);
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    if constexpr (kVector) {
      const int i = column(c, 0);
      if (!live || i >= a.width) continue;
      if (a.residual)
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.residual_out) + row * a.residual_out_stride + i) =
            narrow8(h[c], r_bf16);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[c][e] = h[c][e] * f * (w[c][e] + a.weight_offset);
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + row * a.out_stride + i) =
          narrow8(h[c], a.out_type == TRIS_DTYPE_BF16);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int i = column(c, e);
        if (!live || i >= a.width) continue;
        if (a.residual) store1(a.residual_out, row * a.residual_out_stride + i, h[c][e], a.residual_type);
        store1(a.out, row * a.out_stride + i, h[c][e] * f * (w[c][e] + a.weight_offset), a.out_type);
      }
    }
  }
}

template <int kLanes, int kChunks>
static void rms_norm_launch(const RmsNormArgs& a, bool vector, hipStream_t st) {
  constexpr int kRows = kLanes <= kWave ? 256 / kLanes : 1;
  const dim3 grid(static_cast<unsigned>((a.rows + kRows - 1) / kRows)), block(kLanes <= kWave ? 256 : kLanes);
  if (vector) hipLaunchKernelGGL((rms_norm_kernel<kLanes, kChunks, true>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((rms_norm_kernel<kLanes, kChunks, false>), grid, block, 0, st, a);
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
  bool vector = width % 8 == 0 && aligned16(x) && aligned16(weight) && aligned16(out) && aligned16(residual) &&
                aligned16(residual_out);
  if (rows > 1)
    for (const int64_t v : {x_stride, out_stride, residual_stride, residual_out_stride}) vector = vector && v % 8 == 0;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (width <= 64) rms_norm_launch<8, 1>(a, vector, st);
  else if (width <= 128) rms_norm_launch<16, 1>(a, vector, st);
  else if (width <= 256) rms_norm_launch<32, 1>(a, vector, st);
  else if (width <= 512) rms_norm_launch<64, 1>(a, vector, st);
  else if (width <= 1024) rms_norm_launch<64, 2>(a, vector, st);
  else if (width <= 2048) rms_norm_launch<256, 1>(a, vector, st);
  else if (width <= 4096) rms_norm_launch<256, 2>(a, vector, st);
  else if (width <= 8192) rms_norm_launch<512, 2>(a, vector, st);
  else if (width <= 16384) rms_norm_launch<1024, 2>(a, vector, st);
  else rms_norm_launch<1024, 4>(a, vector, st);
  return check_launch(who);
}
