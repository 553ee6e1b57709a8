// The paged key / value cache: host checks and addressing shared by the append and the attention.
#pragma once

#include <algorithm>
#include <array>

#include "tris_dtype.h"

namespace tris {

constexpr float kE4m3Max = 448.0f;
constexpr float kSmallestScale = 1.17549435e-38f;  // 2^-126

// Positions that a sequence's row of the block table can address (the entry checks keep it below 2^31 - 2^16, so that a
// few tiles past the end are still int32).
__host__ __device__ inline int32_t cache_positions(const tris_paged_cache& c) { return c.max_pages * c.page_size; }

// Division of positions (below 2^31) by the page size d: x / d = x * m >> (31 + e), 2^e >= d, m = 2^(31 + e) / d + 1,
// exact since m d - 2^(31 + e) <= 2^e.
struct PageDivision {
  uint32_t magic, shift;
  explicit PageDivision(int32_t d) {
    uint32_t e = 0;
    while ((1u << e) < static_cast<uint32_t>(d)) ++e;
    magic = static_cast<uint32_t>((1ull << (31 + e)) / static_cast<uint32_t>(d) + 1);
    shift = 31 + e;
  }
  __device__ int operator()(int x) const {
    return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(x)) * magic) >> shift);
  }
};

// Whether rows of `dim` values over these dimensions (sizes and strides) share no memory: each dimension's stride is past
// all that the ones of smaller strides span.
struct RowDimension {
  int64_t size, stride;
};
template <size_t kDims>
bool rows_apart(std::array<RowDimension, kDims> dims, int64_t dim) {
  std::sort(dims.begin(), dims.end(), [](const RowDimension& x, const RowDimension& y) { return x.stride < y.stride; });
  __int128 span = dim;
  for (const RowDimension& d : dims) {
    if (d.size <= 1) continue;
    if (d.stride < span) return false;
    span += static_cast<__int128>(d.size - 1) * d.stride;
  }
  return true;
}

// The cache's own contract; `who` names the entry point in the message.
inline int check_paged_cache(const char* who, const tris_paged_cache* c, int32_t act_type) {
  TRIS_REQUIRE(c != nullptr, "%s: null cache", who);
  TRIS_REQUIRE(c->batch >= 0 && c->num_pages >= 1 && c->kv_heads >= 1 && c->max_pages >= 0,
               "%s: a cache has at least one page and one head", who);
  TRIS_REQUIRE(c->page_size >= 1, "%s: page_size must be positive", who);
  TRIS_REQUIRE(c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256, "%s: head_dim must be 64, 128 or 256",
               who);
  TRIS_REQUIRE(is_16bit(act_type), "%s: activations must be fp16 or bf16", who);
  const bool e4m3 = c->dtype == TRIS_DTYPE_E4M3;
  TRIS_REQUIRE(e4m3 || c->dtype == act_type, "%s: the cache must be e4m3 or of the activations' type", who);
  TRIS_REQUIRE(e4m3 == (c->k_scale != nullptr) && e4m3 == (c->v_scale != nullptr),
               "%s: an e4m3 cache, and no other, has k_scale and v_scale", who);
  TRIS_REQUIRE(c->batch == 0 || (c->k && c->v && c->seq_lens && (c->block_table || c->max_pages == 0)),
               "%s: null pointer", who);
  TRIS_REQUIRE(static_cast<int64_t>(c->max_pages) * c->page_size < (1LL << 31) - (1 << 16),
               "%s: block table too wide", who);
  TRIS_REQUIRE(c->table_stride >= 0, "%s: negative table stride", who);
  const int size = e4m3 ? 1 : 2;
  for (const int64_t s : {c->k_page_stride, c->k_head_stride, c->k_slot_stride, c->v_page_stride, c->v_head_stride,
                          c->v_slot_stride})
    TRIS_REQUIRE(s >= 0 && s * size % 16 == 0, "%s: cache rows must be 16-byte aligned", who);
  TRIS_REQUIRE(aligned16(c->k) && aligned16(c->v), "%s: cache rows must be 16-byte aligned", who);
  // (a page's bytes along its slots are int32 in the kernels)
  const auto slots_fit = [&](int64_t stride, int bytes) {
    return stride >= 0 && stride <= ((1LL << 31) - 1) / bytes / c->page_size;
  };
  TRIS_REQUIRE(slots_fit(c->k_slot_stride, size) && slots_fit(c->v_slot_stride, size) &&
                   (!e4m3 || (slots_fit(c->k_scale_slot_stride, 4) && slots_fit(c->v_scale_slot_stride, 4))),
               "%s: slot stride too large", who);
  TRIS_REQUIRE(c->page_size == 1 || (c->k_slot_stride >= c->head_dim && c->v_slot_stride >= c->head_dim),
               "%s: cache rows overlap", who);
  for (const int64_t s : {c->k_scale_page_stride, c->k_scale_head_stride, c->v_scale_page_stride,
                          c->v_scale_head_stride})
    TRIS_REQUIRE(!e4m3 || s >= 0, "%s: negative scale stride", who);
  return TRIS_OK;
}

// What a cache that is written to has to be: pages, heads and slots without shared memory; its scales likewise.
inline bool cache_rows_apart(const tris_paged_cache& c, int64_t page, int64_t head, int64_t slot, int64_t row) {
  return rows_apart<3>({{{c.num_pages, page}, {c.kv_heads, head}, {c.page_size, slot}}}, row);
}
inline bool cache_rows_apart(const tris_paged_cache& c) {
  return cache_rows_apart(c, c.k_page_stride, c.k_head_stride, c.k_slot_stride, c.head_dim) &&
         cache_rows_apart(c, c.v_page_stride, c.v_head_stride, c.v_slot_stride, c.head_dim);
}
inline bool cache_scales_apart(const tris_paged_cache& c) {
  return !c.k_scale || (cache_rows_apart(c, c.k_scale_page_stride, c.k_scale_head_stride, c.k_scale_slot_stride, 1) &&
                        cache_rows_apart(c, c.v_scale_page_stride, c.v_scale_head_stride, c.v_scale_slot_stride, 1));
}

// Whether two pools of rows of `row` bytes, `to` bytes from the first's beginning to the second's, share no memory, by their
// strides (in bytes, largest first, each pool's own rows apart).  Parts of one buffer may interleave: under the same largest
// stride P a unit of the second meets no units of the first but those `to` mod P and `to` mod P - P bytes from it, since no
// unit is longer than P.  Pools whose strides differ before the ones' units end up beside the others' are taken as shared.
template <size_t kDims>
bool pools_apart(const std::array<RowDimension, kDims>& x, const std::array<RowDimension, kDims>& y, size_t from,
                 __int128 to, int64_t row) {
  __int128 x_end = row, y_end = to + row;
  for (size_t i = from; i < kDims; ++i) {
    x_end += static_cast<__int128>(x[i].size - 1) * x[i].stride;
    y_end += static_cast<__int128>(y[i].size - 1) * y[i].stride;
  }
  if (to >= x_end || y_end <= 0) return true;
  if (from == kDims || x[from].stride != y[from].stride) return false;
  const __int128 step = x[from].stride;
  if (step == 0) return false;  // (a dimension of one, and those behind it)
  const __int128 rest = (to % step + step) % step;
  return pools_apart(x, y, from + 1, rest, row) && pools_apart(x, y, from + 1, rest - step, row);
}

// The cache's keys and values, and their scales, for a call that moves both at the same time.
inline bool keys_and_values_apart(const tris_paged_cache& c) {
  const auto apart = [&c](const void* k, std::array<int64_t, 3> k_strides, const void* v, std::array<int64_t, 3> v_strides,
                          int64_t values, int64_t bytes) {
    const auto dims = [&](const std::array<int64_t, 3>& strides) {
      const int32_t sizes[3] = {c.num_pages, c.kv_heads, c.page_size};
      std::array<RowDimension, 3> d;
      for (int i = 0; i < 3; ++i) d[i] = RowDimension{sizes[i], sizes[i] > 1 ? strides[i] * bytes : 0};
      std::sort(d.begin(), d.end(), [](const RowDimension& x, const RowDimension& y) { return x.stride > y.stride; });
      return d;
    };
    const __int128 to = static_cast<__int128>(reinterpret_cast<uintptr_t>(v)) - reinterpret_cast<uintptr_t>(k);
    return pools_apart<3>(dims(k_strides), dims(v_strides), 0, to, values * bytes);
  };
  return apart(c.k, {c.k_page_stride, c.k_head_stride, c.k_slot_stride}, c.v,
               {c.v_page_stride, c.v_head_stride, c.v_slot_stride}, c.head_dim, c.dtype == TRIS_DTYPE_E4M3 ? 1 : 2) &&
         (!c.k_scale ||
          apart(c.k_scale, {c.k_scale_page_stride, c.k_scale_head_stride, c.k_scale_slot_stride}, c.v_scale,
                {c.v_scale_page_stride, c.v_scale_head_stride, c.v_scale_slot_stride}, 1, 4));
}

// Sums of attention weights, a row of all positions for each (sequence, kv head): strides that keep the rows apart.
inline bool sum_rows_apart(const tris_paged_cache& c, int64_t seq_stride, int64_t head_stride) {
  return seq_stride >= 0 && head_stride >= 0 &&
         rows_apart<2>({{{c.batch, seq_stride}, {c.kv_heads, head_stride}}}, cache_positions(c));
}

}  // namespace tris
