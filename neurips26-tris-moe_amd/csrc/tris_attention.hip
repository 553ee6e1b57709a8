// Attention of one new token a sequence over the paged cache.
//
//   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  s_j = scale * q . k_j,  m = max_j s_j
//
// One pass with the running maximum and sum: a workgroup has one query head, its wavefronts take keys in turn, a lane
// holds head_dim / 64 values.
#include "tris_paged.h"

namespace tris {

struct AttentionArgs {
  const uint16_t* q;
  uint16_t* out;
  int64_t q_seq, q_head, out_seq, out_head;
  float scale;
  int32_t window, q_heads, bf16;
  tris_paged_cache c;
};

__device__ __forceinline__ float e4m3_to_f32(uint32_t b) { return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(b), 0); }

template <int kPer>
__global__ __launch_bounds__(256) void attention_decode_kernel(const AttentionArgs a) {
  constexpr int kDim = kPer * kWave;
  __shared__ float sh_m[4], sh_l[4], sh_o[4][kDim];
  const int b = blockIdx.x / a.q_heads, h = blockIdx.x % a.q_heads;
  const int kvh = h / (a.q_heads / a.c.kv_heads);
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const bool e4m3 = a.c.dtype == TRIS_DTYPE_E4M3;
  const int n = min(max(a.c.seq_lens[b], 0), cache_positions(a.c));
  const int first = a.window > 0 ? max(0, n - a.window) : 0;
  const int type = a.bf16 ? TRIS_DTYPE_BF16 : TRIS_DTYPE_F16;
  float q[kPer], o[kPer], m = -INFINITY, l = 0.0f;
  for (int i = 0; i < kPer; ++i) {
    q[i] = load1(a.q, b * a.q_seq + h * a.q_head + lane * kPer + i, type);
    o[i] = 0.0f;
  }
  for (int j = first + wave; j < n; j += 4) {
    const int page = a.c.block_table[b * a.c.table_stride + j / a.c.page_size], slot = j % a.c.page_size;
    if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(a.c.num_pages)) continue;
    const int64_t ka = page * a.c.k_page_stride + kvh * a.c.k_head_stride + slot * a.c.k_slot_stride + lane * kPer;
    const int64_t va = page * a.c.v_page_stride + kvh * a.c.v_head_stride + slot * a.c.v_slot_stride + lane * kPer;
    float s = 0.0f, v[kPer], ks = 1.0f, vs = 1.0f;
    if (e4m3) {
      ks = a.c.k_scale[page * a.c.k_scale_page_stride + kvh * a.c.k_scale_head_stride + slot * a.c.k_scale_slot_stride];
      vs = a.c.v_scale[page * a.c.v_scale_page_stride + kvh * a.c.v_scale_head_stride + slot * a.c.v_scale_slot_stride];
    }
    for (int i = 0; i < kPer; ++i) {
      const float k = e4m3 ? e4m3_to_f32(static_cast<const uint8_t*>(a.c.k)[ka + i]) : load1(a.c.k, ka + i, type);
      v[i] = (e4m3 ? e4m3_to_f32(static_cast<const uint8_t*>(a.c.v)[va + i]) : load1(a.c.v, va + i, type)) * vs;
      s += q[i] * k;
    }
    s = wave_sum_f32(s) * ks * a.scale;
    const float now = fmaxf(m, s), keep = now == -INFINITY ? 0.0f : now;
    const float f = expf(m - keep), p = expf(s - keep);
    l = l * f + p;
    for (int i = 0; i < kPer; ++i) o[i] = o[i] * f + p * v[i];
    m = now;
  }
  if (lane == 0) {
    sh_m[wave] = m;
    sh_l[wave] = l;
  }
  for (int i = 0; i < kPer; ++i) sh_o[wave][lane * kPer + i] = o[i];
  __syncthreads();
  float most = fmaxf(fmaxf(sh_m[0], sh_m[1]), fmaxf(sh_m[2], sh_m[3]));
  if (most == -INFINITY) most = 0.0f;
  float total = 0.0f;
  for (int w = 0; w < 4; ++w) total += sh_l[w] * expf(sh_m[w] - most);
  for (int d = threadIdx.x; d < kDim; d += 256) {
    float y = 0.0f;
    for (int w = 0; w < 4; ++w) y += sh_o[w][d] * expf(sh_m[w] - most);
    store1(a.out, b * a.out_seq + h * a.out_head + d, total == 0.0f ? 0.0f : y / total, type);
  }
}

}  // namespace tris

using namespace tris;

extern "C" int64_t tris_paged_attention_workspace_bytes(int32_t batch, int32_t q_heads, int32_t kv_heads,
                                                        int32_t head_dim, int32_t max_pages, int32_t page_size) {
  return 0;
}

extern "C" int tris_paged_attention_decode(const void* q, int64_t q_seq_stride, int64_t q_head_stride, int32_t q_type,
                                           int32_t q_heads, const tris_paged_cache* cache, float scale, int32_t window,
                                           void* out, int64_t out_seq_stride, int64_t out_head_stride, void* workspace,
                                           int64_t workspace_bytes, void* stream) {
  const char* who = "tris_paged_attention_decode";
  if (const int rc = check_paged_cache(who, cache, q_type)) return rc;
  TRIS_REQUIRE(q_heads >= 1 && q_heads % cache->kv_heads == 0, "%s: q_heads must be a multiple of kv_heads", who);
  TRIS_REQUIRE(window >= 0, "%s: negative window", who);
  if (cache->batch == 0) return TRIS_OK;
  TRIS_REQUIRE(q && out, "%s: null pointer", who);
  for (const int64_t s : {q_seq_stride, q_head_stride, out_seq_stride, out_head_stride})
    TRIS_REQUIRE(s >= 0 && s % 8 == 0, "%s: rows must be 16-byte aligned", who);
  TRIS_REQUIRE(aligned16(q) && aligned16(out), "%s: rows must be 16-byte aligned", who);
  const int64_t blocks = static_cast<int64_t>(cache->batch) * q_heads;
  TRIS_REQUIRE(blocks <= 2147483647LL, "%s: too many rows", who);
  AttentionArgs a{static_cast<const uint16_t*>(q), static_cast<uint16_t*>(out), q_seq_stride, q_head_stride,
                  out_seq_stride, out_head_stride, scale, window, q_heads, q_type == TRIS_DTYPE_BF16, *cache};
  const dim3 grid(static_cast<unsigned>(blocks)), block(256);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (cache->head_dim == 64) hipLaunchKernelGGL(attention_decode_kernel<1>, grid, block, 0, st, a);
  else if (cache->head_dim == 128) hipLaunchKernelGGL(attention_decode_kernel<2>, grid, block, 0, st, a);
  else hipLaunchKernelGGL(attention_decode_kernel<4>, grid, block, 0, st, a);
  return check_launch(who);
}
