// Root-mean-square norm with the residual's addition.
//
//   h = x + residual,  residual_out = round(h),  out = round(h * rsqrt(mean(h^2) + eps) * (weight + offset))
//
// Everything between the loads and the one rounding of each output is fp32; the sum of squares of a row is a fixed
// tree for its width, so results do not depend on the other rows.
//
// Bound by memory: four 16-bit values a column with a residual.  In a graph, bf16: 8192 x 4096 with the residual (268 MB)
// 42 us, 6.3 TB/s, above a copy's 5.2 since part of it stays in the memory-side cache; 10656 x 128 3.8 us; one row of
// 4096 2.8 us, a launch's own time.  A width that eight does not divide costs its unaligned rows: 8192 x 4095 66 us (132
// one value at a time).
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

// Eight 16-bit values at column i of a row that is `width` long.  Rows need no alignment: the copies are 16-byte accesses
// whatever the address, which this GPU's global memory takes.  kTail: the row's last run may be shorter.
template <bool kTail>
__device__ __forceinline__ uint4 load_run(const void* p, int64_t at, int i, int width) {
  const uint16_t* src = static_cast<const uint16_t*>(p) + at + i;
  uint4 v = {0, 0, 0, 0};
  if (!kTail || i + 8 <= width) {
    __builtin_memcpy(&v, src, 16);
  } else {
    uint32_t u[4] = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (i + e < width) u[e / 2] |= static_cast<uint32_t>(src[e]) << (e % 2 * 16);
    v = make_uint4(u[0], u[1], u[2], u[3]);
  }
  return v;
}
template <bool kTail>
__device__ __forceinline__ void store_run(void* p, int64_t at, int i, int width, const uint4 v) {
  uint16_t* dst = static_cast<uint16_t*>(p) + at + i;
  if (!kTail || i + 8 <= width) {
    __builtin_memcpy(dst, &v, 16);
  } else {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (i + e < width) dst[e] = static_cast<uint16_t>(u[e / 2] >> (e % 2 * 16));
  }
}

// kLanes threads a row, each with kChunks runs of eight columns in registers, so that a row is read once.  Up to 64
// lanes a row, so to 1024 columns, a workgroup has 256 / kLanes rows and a row's sum stays in its wavefront; above, a row
// has the workgroup.
// Measured with the residual: 10656 x 64 and x 128, as many lanes as runs 3.06 / 3.76 us, a wavefront a row 5.25 / 5.44;
// 4096 columns, a workgroup of 256 for 8192 rows 42.2 us and for one 2.7, a wavefront a row 44.2 and 4.4, 128 threads
// 43.0 and 3.3; 8192 columns, 512 threads 42.1 / 2.95, 1024 44.5 / 3.05, 256 42.9 / 3.4.  1024 columns, a wavefront for
// 8192 rows 11.2 and for one 2.5, 128 threads 12.4 and 2.35; 2048, 256 threads 23.5 and 2.4, 128 23.5 and 2.65, a wavefront
// 23.8 and 3.4; 16384, 1024 threads for 2048 rows 45.6 and for one 3.6, 512 46.3 and 4.1; 32768, 1024 threads for 1024 rows
// 51.8 and for one 5.1, 512 54.5 and 6.1.
template <int kLanes, int kChunks, bool kTail>
__global__ __launch_bounds__(kLanes > 256 ? kLanes : 256) void rms_norm_kernel(const RmsNormArgs a) {
  constexpr int kRows = kLanes <= kWave ? 256 / kLanes : 1;
  const int t = threadIdx.x % kLanes;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / kLanes;
  const bool live = row < a.rows, r_bf16 = a.residual_type == TRIS_DTYPE_BF16, w_f32 = a.weight_type == TRIS_DTYPE_F32;
  // the row and the weights in flight together
  uint4 xs[kChunks], rs[kChunks], ws[kChunks];
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    const int i = (c * kLanes + t) * 8;
    if (!live || i >= a.width) continue;
    xs[c] = load_run<kTail>(a.x, row * a.x_stride, i, a.width);
    if (a.residual) rs[c] = load_run<kTail>(a.residual, row * a.residual_stride, i, a.width);
    if (!w_f32) ws[c] = load_run<kTail>(a.weight, 0, i, a.width);
  }
  float h[kChunks][8], sq = 0.0f;
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    if (!live || (c * kLanes + t) * 8 >= a.width) continue;
    widen8(xs[c], a.x_type == TRIS_DTYPE_BF16, h[c]);
    if (a.residual) {
      float r[8];
      widen8(rs[c], r_bf16, r);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[c][e] += r[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) sq += h[c][e] * h[c][e];
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
    const int i = (c * kLanes + t) * 8;
    if (!live || i >= a.width) continue;
    if (a.residual) store_run<kTail>(a.residual_out, row * a.residual_out_stride, i, a.width, narrow8(h[c], r_bf16));
    float w[8];
    if (w_f32) {
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = !kTail || i + e < a.width ? static_cast<const float*>(a.weight)[i + e] : 0.0f;
    } else {
      widen8(ws[c], a.weight_type == TRIS_DTYPE_BF16, w);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = h[c][e] * f * (w[e] + a.weight_offset);
    store_run<kTail>(a.out, row * a.out_stride, i, a.width, narrow8(w, a.out_type == TRIS_DTYPE_BF16));
  }
}

template <int kLanes, int kChunks>
static int rms_norm_launch(const char* who, const RmsNormArgs& a, hipStream_t st) {
  constexpr int kRows = kLanes <= kWave ? 256 / kLanes : 1, kThreads = kLanes <= kWave ? 256 : kLanes;
  const int64_t blocks = (a.rows + kRows - 1) / kRows;
  TRIS_REQUIRE(blocks * kThreads < 1LL << 32, "%s: too many rows", who);  // of one launch
  const dim3 grid(static_cast<unsigned>(blocks)), block(kThreads);
  if (a.width % 8 == 0) hipLaunchKernelGGL((rms_norm_kernel<kLanes, kChunks, false>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((rms_norm_kernel<kLanes, kChunks, true>), grid, block, 0, st, a);
  return check_launch(who);
}

}  // namespace tris

using namespace tris;

extern "C" int tris_rms_norm(const void* x, int32_t x_type, int64_t x_stride, const void* residual,
                             int32_t residual_type, int64_t residual_stride, const void* weight, int32_t weight_type,
                             float weight_offset, float eps, int64_t rows, int32_t width, void* out, int32_t out_type,
                             int64_t out_stride, void* residual_out, int64_t residual_out_stride, void* stream) {
  const char* who = "tris_rms_norm";
  TRIS_REQUIRE(rows >= 0 && width >= 1 && width <= 32768, "%s: rows must not be negative, width 1 to 32768", who);
  TRIS_REQUIRE(rows < 1LL << 32, "%s: too many rows", who);
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
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (width <= 64) return rms_norm_launch<8, 1>(who, a, st);
  if (width <= 128) return rms_norm_launch<16, 1>(who, a, st);
  if (width <= 256) return rms_norm_launch<32, 1>(who, a, st);
  if (width <= 512) return rms_norm_launch<64, 1>(who, a, st);
  if (width <= 1024) return rms_norm_launch<64, 2>(who, a, st);
  if (width <= 2048) return rms_norm_launch<256, 1>(who, a, st);
  if (width <= 4096) return rms_norm_launch<256, 2>(who, a, st);
  if (width <= 8192) return rms_norm_launch<512, 2>(who, a, st);
  if (width <= 16384) return rms_norm_launch<1024, 2>(who, a, st);
  return rms_norm_launch<1024, 4>(who, a, st);
}
