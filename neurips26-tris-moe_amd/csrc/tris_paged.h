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

}  // namespace tris
