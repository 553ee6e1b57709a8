// Rotation of queries and keys by their positions, and the append of keys and values to the paged cache.
//
// One launch does the three tensors.  A thread has 16 of a head's values: in a rotated part eight of the lower half and
// the eight that pair with them, elsewhere sixteen in a row.  A wavefront has up to kUnits times 64 such units of one
// token: all their values are in flight while the token's position, page and table row are looked up, once for all,
// and so are the cosines and sines, since a lane has the same part of each of its heads.  An 8-bit row's largest
// magnitude is a maximum over the head's head_dim / 16 neighbouring lanes.
//
// Bound by memory where there are many tokens: 8189 of 32 query and 8 kv heads of 128, bf16 (205 MB), 42.8 us in a graph over
// three states, 4.8 TB/s (a large copy 5.15); else by two memory latencies (boundaries and lengths, then page and angles): one
// token for each of 16 sequences 3.5 us.  With positions of their own, on three axes, 42.3 and 4.2 us, in turn with these.
#include "tris_paged.h"

// The rotation's two products and their sum are rounded one by one, as the same torch expression rounds them, so that
// the values (and the 8-bit elements made of them) do not depend on which of the two wrote a cache.
#pragma clang fp contract(off)

namespace tris {

constexpr int kMaxAxes = TRIS_MAX_ROTARY_AXES;
constexpr int kMostPairs = 128;  // of the widest head

struct AppendArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* q_out;
  const float* cos;
  const float* sin;
  const int32_t* query_start;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, qo_token, qo_head;
  int32_t act_bf16, tokens, q_heads, rotary_dim, zero_unplaced, token_waves;
  PageDivision page_of;
  const int32_t* token_positions;  // [axes][tokens], rows axis_stride apart
  int64_t axis_stride;
  int32_t axes, interleaved, table_rows;
  int32_t ends[kMaxAxes];  // of the axes' pairs: the first pair past them
  tris_paged_cache c;
};

// The axis whose position turns pair i: sections one after the other, or, interleaved, the axes in turn while they have
// pairs left and then the first.
__device__ __forceinline__ int pair_axis(const AppendArgs& a, int i) {
  if (a.interleaved) {
    const int axis = i % a.axes;
    return i < a.ends[axis] ? axis : 0;
  }
  int axis = 0;
#pragma unroll
  for (int n = 0; n < kMaxAxes - 1; ++n) axis += n < a.axes - 1 && i >= a.ends[n];
  return axis;
}

// The sequence whose new tokens hold token t, or -1; *pos: the token's position.  The wavefront reads 64 boundaries and
// lengths at a time and takes the first boundary past t.
__device__ __forceinline__ int token_sequence(const AppendArgs& a, int t, int64_t* pos) {
  if (a.query_start == nullptr) {
    if (t >= a.c.batch) return -1;
    *pos = static_cast<int64_t>(a.c.seq_lens[t]) - 1;
    return t;
  }
  const int lane = threadIdx.x % kWave, begin = a.query_start[0];
  for (int b0 = 0; b0 < a.c.batch; b0 += kWave) {
    const int b = b0 + lane;
    const int end = b < a.c.batch ? a.query_start[b + 1] : 0, length = b < a.c.batch ? a.c.seq_lens[b] : 0;
    const uint64_t past = __ballot(b < a.c.batch && end > t);
    if (past) {
      const int l = __builtin_ctzll(past);
      *pos = static_cast<int64_t>(__builtin_amdgcn_readlane(length, l)) - (__builtin_amdgcn_readlane(end, l) - t);
      return t >= begin ? b0 + l : -1;
    }
  }
  return -1;
}

// eight values of one row as e4m3: v / scale, round to nearest even
__device__ __forceinline__ uint2 e4m3x8(const float v[8], float scale) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int p = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i] / scale, v[4 * i + 1] / scale, 0, false);
    p = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2] / scale, v[4 * i + 3] / scale, p, true);
    w[i] = static_cast<uint32_t>(p);
  }
  return make_uint2(w[0], w[1]);
}

// 1, 2, 3, 4, 6 units: 8189 tokens 43.0, 40.6, 40.0, 40.6, 44.3 us; one token for each of 16 sequences 3.3, 3.7, 4.3, 4.4,
// 6.0.
constexpr int kUnits = 2;

template <bool kE4m3, bool kAxes>
__global__ __launch_bounds__(256) void rotary_append_kernel(const AppendArgs a) {
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(blockIdx.x) * 4 + static_cast<int>(threadIdx.x) / kWave);
  const int t = wave / a.token_waves;
  if (t >= a.tokens) return;
  const int lane = threadIdx.x % kWave, lanes = a.c.head_dim / 16, half = a.rotary_dim / 2;
  const bool bf16 = a.act_bf16 != 0;
  const int heads = a.q_heads + 2 * a.c.kv_heads;
  const int part = lane % lanes;  // of every head that the lane has
  const int turning = part * 8 < half;
  // columns of the two runs in a query or key, and in a value
  const int lo_qk = turning ? part * 8 : a.rotary_dim + (part - half / 8) * 16, hi_qk = turning ? lo_qk + half : lo_qk + 8;
  const int lo_v = part * 16, hi_v = lo_v + 8;
  const int head0 = (wave - t * a.token_waves) * kWave / lanes + lane / lanes, step = a.token_waves * kWave / lanes;

  uint4 xs[kUnits], ys[kUnits];
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    const int h = head0 + i * step;
    if (h >= heads) continue;
    const bool is_q = h < a.q_heads, is_k = !is_q && h < a.q_heads + a.c.kv_heads;
    const uint16_t* src = is_q   ? a.q + t * a.q_token + h * a.q_head
                          : is_k ? a.k + t * a.k_token + (h - a.q_heads) * a.k_head
                                 : a.v + t * a.v_token + (h - a.q_heads - a.c.kv_heads) * a.v_head;
    xs[i] = *reinterpret_cast<const uint4*>(src + (is_q || is_k ? lo_qk : lo_v));
    ys[i] = *reinterpret_cast<const uint4*>(src + (is_q || is_k ? hi_qk : hi_v));
  }

  constexpr int kPairUnits = kMostPairs / kWave;
  __shared__ float sh_cos[kAxes ? 4 : 1][kMostPairs], sh_sin[kAxes ? 4 : 1][kMostPairs];
  // each pair's angle once for the wavefront, asked for before the token's place is known, handed to the lanes that turn
  // it through LDS (8189 tokens 42.3 us; asked for when the place is known 44.6, with every lane loading its own eight 53.2)
  float pair_cos[kPairUnits] = {}, pair_sin[kPairUnits] = {};
  bool turnable = true;
  if constexpr (kAxes) {
    int at_row[kMaxAxes];
#pragma unroll
    for (int n = 0; n < kMaxAxes; ++n) {
      at_row[n] = n < a.axes ? a.token_positions[n * a.axis_stride + t] : 0;
      turnable = turnable && at_row[n] >= 0 && at_row[n] < a.table_rows;
    }
#pragma unroll
    for (int u = 0; u < kPairUnits; ++u) {
      if (u * kWave >= half) break;
      const int pair = u * kWave + lane, axis = pair_axis(a, pair);
      int row = at_row[0];
#pragma unroll
      for (int n = 1; n < kMaxAxes; ++n) row = axis == n ? at_row[n] : row;
      if (pair < half && turnable) {
        pair_cos[u] = a.cos[static_cast<int64_t>(row) * half + pair];
        pair_sin[u] = a.sin[static_cast<int64_t>(row) * half + pair];
      }
    }
  }

  int64_t place = -1;
  const int seq = token_sequence(a, t, &place);
  const int pos = seq >= 0 && place >= 0 && place < cache_positions(a.c) && turnable ? static_cast<int>(place) : -1;
  int page = -1, slot = 0;
  float cs[8], sn[8];
  if (pos >= 0) {
    const int i = a.page_of(pos);
    page = a.c.block_table[seq * a.c.table_stride + i];
    slot = pos - i * a.c.page_size;
    if constexpr (kAxes) {
#pragma unroll
      for (int u = 0; u < kPairUnits; ++u) {
        if (u * kWave >= half) break;
        sh_cos[threadIdx.x / kWave][u * kWave + lane] = pair_cos[u];
        sh_sin[threadIdx.x / kWave][u * kWave + lane] = pair_sin[u];
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      if (turning) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          cs[e] = sh_cos[threadIdx.x / kWave][lo_qk + e];
          sn[e] = sh_sin[threadIdx.x / kWave][lo_qk + e];
        }
      }
    } else if (turning) {
      const float* c = a.cos + static_cast<int64_t>(pos) * half + lo_qk;
      const float* s = a.sin + static_cast<int64_t>(pos) * half + lo_qk;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        cs[e] = c[e];
        sn[e] = s[e];
      }
    }
    if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(a.c.num_pages)) page = -1;
  }

#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    const int h = head0 + i * step;
    if (h >= heads) continue;
    const bool is_q = h < a.q_heads, is_k = !is_q && h < a.q_heads + a.c.kv_heads;
    const int hh = is_q ? h : is_k ? h - a.q_heads : h - a.q_heads - a.c.kv_heads;
    const int lo = is_q || is_k ? lo_qk : lo_v, hi = is_q || is_k ? hi_qk : hi_v;
    uint16_t* q_out = a.q_out + t * a.qo_token + hh * a.qo_head;
    if (is_q && pos < 0) {
      if (a.zero_unplaced) {
        *reinterpret_cast<uint4*>(q_out + lo) = make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(q_out + hi) = make_uint4(0, 0, 0, 0);
      }
      continue;
    }
    if (!is_q && page < 0) continue;
    float x[8], y[8];
    widen8(xs[i], bf16, x);
    widen8(ys[i], bf16, y);
    if (turning && (is_q || is_k)) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float xe = x[e], ye = y[e];
        x[e] = xe * cs[e] - ye * sn[e];
        y[e] = ye * cs[e] + xe * sn[e];
      }
    }
    const int64_t at = is_k ? page * a.c.k_page_stride + hh * a.c.k_head_stride + slot * a.c.k_slot_stride
                            : page * a.c.v_page_stride + hh * a.c.v_head_stride + slot * a.c.v_slot_stride;
    void* rows = is_k ? a.c.k : a.c.v;
    if (is_q || !kE4m3) {
      uint16_t* o = is_q ? q_out : static_cast<uint16_t*>(rows) + at;
      *reinterpret_cast<uint4*>(o + lo) = narrow8(x, bf16);
      *reinterpret_cast<uint4*>(o + hi) = narrow8(y, bf16);
      continue;
    }
    // magnitudes compare as their bits, and a NaN's are above infinity's, so that one in the row becomes the scale
    uint32_t most = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      most = max(most, __float_as_uint(x[e]) & 0x7FFFFFFFu);
      most = max(most, __float_as_uint(y[e]) & 0x7FFFFFFFu);
    }
    for (int d = 1; d < lanes; d *= 2) most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), d)));
    float scale = __uint_as_float(most) * (1.0f / kE4m3Max);
    if (scale < kSmallestScale) scale = kSmallestScale;
    uint8_t* o = static_cast<uint8_t*>(rows) + at;
    *reinterpret_cast<uint2*>(o + lo) = e4m3x8(x, scale);
    *reinterpret_cast<uint2*>(o + hi) = e4m3x8(y, scale);
    if (part == 0) {
      if (is_k)
        a.c.k_scale[page * a.c.k_scale_page_stride + hh * a.c.k_scale_head_stride + slot * a.c.k_scale_slot_stride] = scale;
      else
        a.c.v_scale[page * a.c.v_scale_page_stride + hh * a.c.v_scale_head_stride + slot * a.c.v_scale_slot_stride] = scale;
    }
  }
}

}  // namespace tris

using namespace tris;

namespace {

// The rotary positions of tokens whose places in the cache do not give them.
struct TokenPositions {
  const int32_t* positions;
  int64_t axis_stride;
  int32_t axes, interleaved;
  const int32_t* sections;
};

int append(const char* who, const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k,
           int64_t k_token_stride, int64_t k_head_stride, const void* v, int64_t v_token_stride, int64_t v_head_stride,
           int32_t act_type, int32_t tokens, int32_t q_heads, const float* cos, const float* sin, int32_t rotary_dim,
           int32_t positions, const int32_t* query_start, const tris_paged_cache* cache, void* q_out,
           int64_t q_out_token_stride, int64_t q_out_head_stride, int32_t zero_unplaced, const TokenPositions* given,
           void* stream) {
  if (const int rc = check_paged_cache(who, cache, act_type)) return rc;
  TRIS_REQUIRE(tokens >= 0 && q_heads >= 0, "%s: negative shape", who);
  TRIS_REQUIRE(query_start || tokens == cache->batch, "%s: without query_start there is one token a sequence", who);
  TRIS_REQUIRE(rotary_dim >= 16 && rotary_dim % 16 == 0 && rotary_dim <= cache->head_dim,
               "%s: rotary_dim must be a multiple of 16 up to head_dim", who);
  if (given) {
    TRIS_REQUIRE(given->axes >= 1 && given->axes <= kMaxAxes && given->sections && given->axis_stride >= 0,
                 "%s: positions have 1 to %d axes, a section for each", who, kMaxAxes);
    int64_t pairs = 0;
    for (int i = 0; i < given->axes; ++i) {
      TRIS_REQUIRE(given->sections[i] >= 0, "%s: negative section", who);
      pairs += given->sections[i];
    }
    TRIS_REQUIRE(pairs == rotary_dim / 2, "%s: the sections must add up to rotary_dim / 2 pairs", who);
    for (int i = 1; i < given->axes && given->interleaved; ++i)
      TRIS_REQUIRE(given->sections[i] == 0 || (given->sections[i] - 1) * given->axes + i < rotary_dim / 2,
                   "%s: interleaved sections that do not fit", who);
    TRIS_REQUIRE(positions >= 1, "%s: cos and sin without rows", who);
  } else {
    TRIS_REQUIRE(positions >= cache_positions(*cache), "%s: cos and sin must cover max_pages * page_size positions",
                 who);
  }
  if (tokens == 0) return TRIS_OK;
  TRIS_REQUIRE(cache->batch > 0, "%s: tokens without sequences", who);
  TRIS_REQUIRE(k && v && cos && sin && (q_heads == 0 || (q && q_out)) && (!given || given->positions),
               "%s: null pointer", who);
  for (const int64_t s : {q_heads ? q_token_stride : 0, q_heads ? q_head_stride : 0, k_token_stride, k_head_stride,
                          v_token_stride, v_head_stride, q_heads ? q_out_token_stride : 0,
                          q_heads ? q_out_head_stride : 0})
    TRIS_REQUIRE(s >= 0 && s % 8 == 0, "%s: rows must be 16-byte aligned", who);
  TRIS_REQUIRE(aligned16(k) && aligned16(v) && aligned16(cos) && aligned16(sin) &&
                   (q_heads == 0 || (aligned16(q) && aligned16(q_out))),
               "%s: rows must be 16-byte aligned", who);
  const int64_t units = (static_cast<int64_t>(q_heads) + 2LL * cache->kv_heads) * (cache->head_dim / 16);
  TRIS_REQUIRE(units < (1 << 24), "%s: too many heads", who);
  const tris_paged_cache& c = *cache;
  TRIS_REQUIRE(q_heads == 0 || rows_apart<2>({{{tokens, q_out_token_stride}, {q_heads, q_out_head_stride}}}, c.head_dim),
               "%s: output rows overlap", who);
  TRIS_REQUIRE(cache_rows_apart(c), "%s: cache rows overlap", who);
  TRIS_REQUIRE(cache_scales_apart(c), "%s: cache scales overlap", who);
  const int64_t token_waves = (units + kUnits * kWave - 1) / (kUnits * kWave);
  const int64_t blocks = (tokens * token_waves + 3) / 4;
  TRIS_REQUIRE(blocks < (1LL << 32) / (4 * kWave), "%s: too many tokens", who);  // a launch has less than 2^32 threads
  AppendArgs a{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v),
               static_cast<uint16_t*>(q_out), cos, sin, query_start, q_token_stride, q_head_stride, k_token_stride,
               k_head_stride, v_token_stride, v_head_stride, q_out_token_stride, q_out_head_stride,
               act_type == TRIS_DTYPE_BF16, tokens, q_heads, rotary_dim, zero_unplaced,
               static_cast<int32_t>(token_waves), PageDivision(cache->page_size), nullptr, 0, 0, 0, 0, {}, *cache};
  if (given) {
    a.token_positions = given->positions;
    a.axis_stride = given->axis_stride;
    a.axes = given->axes;
    a.interleaved = given->interleaved;
    a.table_rows = positions;
    for (int i = 0, end = 0; i < given->axes; ++i) {
      end += given->sections[i];
      a.ends[i] = given->interleaved ? given->axes * given->sections[i] : end;
    }
  }
  const dim3 grid(static_cast<unsigned>(blocks)), block(4 * kWave);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (cache->dtype == TRIS_DTYPE_E4M3) {
    if (given) hipLaunchKernelGGL((rotary_append_kernel<true, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((rotary_append_kernel<true, false>), grid, block, 0, st, a);
  } else {
    if (given) hipLaunchKernelGGL((rotary_append_kernel<false, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((rotary_append_kernel<false, false>), grid, block, 0, st, a);
  }
  return check_launch(who);
}

}  // namespace

extern "C" int tris_rotary_append_paged(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k,
                                        int64_t k_token_stride, int64_t k_head_stride, const void* v,
                                        int64_t v_token_stride, int64_t v_head_stride, int32_t act_type,
                                        int32_t tokens, int32_t q_heads, const float* cos, const float* sin,
                                        int32_t rotary_dim, int32_t positions, const int32_t* query_start,
                                        const tris_paged_cache* cache, void* q_out, int64_t q_out_token_stride,
                                        int64_t q_out_head_stride, int32_t zero_unplaced, void* stream) {
  return append("tris_rotary_append_paged", q, q_token_stride, q_head_stride, k, k_token_stride, k_head_stride, v,
                v_token_stride, v_head_stride, act_type, tokens, q_heads, cos, sin, rotary_dim, positions, query_start,
                cache, q_out, q_out_token_stride, q_out_head_stride, zero_unplaced, nullptr, stream);
}

extern "C" int tris_rotary_axes_append_paged(const void* q, int64_t q_token_stride, int64_t q_head_stride,
                                             const void* k, int64_t k_token_stride, int64_t k_head_stride,
                                             const void* v, int64_t v_token_stride, int64_t v_head_stride,
                                             int32_t act_type, int32_t tokens, int32_t q_heads, const float* cos,
                                             const float* sin, int32_t rotary_dim, int32_t positions,
                                             const int32_t* query_start, const tris_paged_cache* cache, void* q_out,
                                             int64_t q_out_token_stride, int64_t q_out_head_stride,
                                             int32_t zero_unplaced, const int32_t* token_positions,
                                             int64_t axis_stride, int32_t axes, const int32_t* sections,
                                             int32_t interleaved, void* stream) {
  const TokenPositions given{token_positions, axis_stride, axes, interleaved != 0, sections};
  return append("tris_rotary_axes_append_paged", q, q_token_stride, q_head_stride, k, k_token_stride, k_head_stride, v,
                v_token_stride, v_head_stride, act_type, tokens, q_heads, cos, sin, rotary_dim, positions, query_start,
                cache, q_out, q_out_token_stride, q_out_head_stride, zero_unplaced, &given, stream);
}
