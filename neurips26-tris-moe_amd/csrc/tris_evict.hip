// Eviction from the paged cache by accumulated attention weight: which positions stay, and the move of what they hold.
//
// Two launches.  The first has a workgroup for each (sequence, kv head): it finds the weight at the border, the
// (budget - sink - recent)-th largest between the first `sink` and the last `recent` positions, digit by digit of a key that
// orders the weights, and lists the positions that stay, in order.  The second moves their rows down in place.
#include "tris_paged.h"

namespace tris {

struct EvictArgs {
  float* sums;
  int64_t sum_seq, sum_head;
  int32_t budget, limit, sink, recent;
  int32_t* new_lens;
  int32_t* kept;
  PageDivision page_of;
  tris_paged_cache c;
};

constexpr int kSelectThreads = 1024;
constexpr int kSelectWaves = kSelectThreads / kWave;

// A weight as an unsigned number of the same order: NaN above all, the zeros equal.
__device__ __forceinline__ uint32_t order_key(float w) {
  if (w != w) return 0xFFFFFFFFu;
  const uint32_t u = __float_as_uint(w == 0.0f ? 0.0f : w);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int evict_length(const EvictArgs& a, int b) {
  return min(max(a.c.seq_lens[b], 0), cache_positions(a.c));
}

__global__ __launch_bounds__(kSelectThreads) void evict_select_kernel(const EvictArgs a) {
  __shared__ int hist[256];
  __shared__ int totals[kSelectWaves];
  __shared__ int pick, above;
  const int row = blockIdx.x, b = row / a.c.kv_heads, h = row - b * a.c.kv_heads;
  const int thread = threadIdx.x, lane = thread % kWave, wave = thread / kWave;
  const int n = evict_length(a, b);
  int32_t* kept = a.kept + static_cast<int64_t>(row) * a.budget;
  bool due = n > a.limit;
  if (due) {
    const int32_t* table = a.c.block_table + b * a.c.table_stride;
    bool good = true;
    for (int i = thread; i <= a.page_of(n - 1); i += kSelectThreads)
      good = good && static_cast<uint32_t>(table[i]) < static_cast<uint32_t>(a.c.num_pages);
    due = __syncthreads_and(good);
  }
  if (h == 0 && thread == 0) a.new_lens[b] = due ? a.budget : a.c.seq_lens[b];
  if (!due) {
    for (int i = thread; i < a.budget; i += kSelectThreads) kept[i] = -1;
    return;
  }
  const float* sums = a.sums + b * a.sum_seq + h * a.sum_head;
  const int lo = a.sink, hi = n - a.recent, want = a.budget - a.sink - a.recent;
  // the key of the want-th largest between lo and hi, and how many of those equal to it stay
  uint32_t border = 0xFFFFFFFFu;
  int equal = 0;
  if (want > 0) {
    uint32_t prefix = 0;
    int left = want;
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (thread < 256) hist[thread] = 0;
      __syncthreads();
      for (int i = lo + thread; i < hi; i += kSelectThreads) {
        const uint32_t key = order_key(sums[i]);
        if (shift == 24 || key >> (shift + 8) == prefix) atomicAdd(&hist[key >> shift & 255], 1);
      }
      __syncthreads();
      if (wave == 0) {
        // four digits a lane, from the largest down
        int c[4], sum = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum += c[i] = hist[255 - (lane * 4 + i)];
        int before = wave_incl_sum_i32(sum) - sum;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (before < left && before + c[i] >= left) {
            pick = 255 - (lane * 4 + i);
            above = before;
          }
          before += c[i];
        }
      }
      __syncthreads();
      prefix = prefix << 8 | static_cast<uint32_t>(pick);
      left -= above;
      __syncthreads();
    }
    border = prefix;
    equal = left;
  }
  // the positions in order: each thread's flags, the waves' counts, the places before
  int placed = 0, ties = 0;
  for (int i0 = 0; i0 < n; i0 += kSelectThreads) {
    const int i = i0 + thread;
    const bool held = i < n && (i < lo || i >= hi);
    bool stays = held, tie = false;
    if (want > 0 && i < n && !held) {
      const uint32_t key = order_key(sums[i]);
      stays = key > border;
      tie = key == border;
    }
    const uint64_t tied = __ballot(tie), below = (1ull << lane) - 1;
    if (lane == 0) totals[wave] = __popcll(tied);
    __syncthreads();
    int rank = ties + __popcll(tied & below);
    for (int w = 0; w < kSelectWaves; ++w) {
      const int t = totals[w];
      rank += w < wave ? t : 0;
      ties += t;
    }
    __syncthreads();
    stays = stays || (tie && rank < equal);
    const uint64_t staying = __ballot(stays);
    if (lane == 0) totals[wave] = __popcll(staying);
    __syncthreads();
    int place = placed + __popcll(staying & below);
    for (int w = 0; w < kSelectWaves; ++w) {
      const int t = totals[w];
      place += w < wave ? t : 0;
      placed += t;
    }
    __syncthreads();
    if (stays) kept[place] = i;
  }
}

// Moves the units of the positions that stay to their places, in place: a workgroup has a slice of every row of one
// (sequence, kv head), so that no other reads what it writes.  It takes them in runs from the first place on: a place is
// never past where its unit comes from, so what a run writes no later run reads, and its own units are in registers
// before any is written.  at(position): a unit's address.
constexpr int kMoveThreads = 1024;
constexpr int kMoveUnits = 4;

template <typename T, typename At>
__device__ __forceinline__ void move_units(const int32_t* kept, int budget, int lanes, At at) {
  const int thread = threadIdx.x, rows = kMoveThreads / lanes, unit = thread % lanes;
  for (int i0 = 0; i0 < budget; i0 += rows * kMoveUnits) {
    T x[kMoveUnits];
    int from[kMoveUnits];
#pragma unroll
    for (int u = 0; u < kMoveUnits; ++u) {
      const int i = i0 + u * rows + thread / lanes;
      from[u] = i < budget ? kept[i] : -1;
      if (from[u] >= 0) x[u] = at(from[u])[unit];
    }
    // every load of the run has arrived before any wavefront stores
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kMoveUnits; ++u) {
      const int i = i0 + u * rows + thread / lanes;
      if (from[u] >= 0 && from[u] != i) at(i)[unit] = x[u];
    }
  }
}

constexpr int kSliceBytes = 64;

__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(const EvictArgs a, int slices, int parts) {
  const int row = blockIdx.x / parts, part = blockIdx.x - row * parts;
  const int b = row / a.c.kv_heads, h = row - b * a.c.kv_heads;
  const int32_t* kept = a.kept + static_cast<int64_t>(row) * a.budget;
  if (kept[0] < 0) return;
  const tris_paged_cache& c = a.c;
  const int32_t* table = c.block_table + b * c.table_stride;
  if (part < 2 * slices) {
    const bool is_v = part >= slices;
    const int size = c.dtype == TRIS_DTYPE_E4M3 ? 1 : 2;
    const int64_t page_bytes = (is_v ? c.v_page_stride : c.k_page_stride) * size;
    const int64_t slot_bytes = (is_v ? c.v_slot_stride : c.k_slot_stride) * size;
    char* base = static_cast<char*>(is_v ? c.v : c.k) + (is_v ? c.v_head_stride : c.k_head_stride) * size * h +
                 (part - (is_v ? slices : 0)) * kSliceBytes;
    move_units<uint4>(kept, a.budget, kSliceBytes / 16, [&](int i) {
      const int p = a.page_of(i);
      return reinterpret_cast<uint4*>(base + table[p] * page_bytes + (i - p * c.page_size) * slot_bytes);
    });
  } else if (part == 2 * slices) {
    float* sums = a.sums + b * a.sum_seq + h * a.sum_head;
    move_units<float>(kept, a.budget, 1, [&](int i) { return sums + i; });
    __syncthreads();
    for (int i = a.budget + threadIdx.x, n = evict_length(a, b); i < n; i += kMoveThreads) sums[i] = 0.0f;
  } else {
    const bool is_v = part == 2 * slices + 2;
    const int64_t page_stride = is_v ? c.v_scale_page_stride : c.k_scale_page_stride;
    const int64_t slot_stride = is_v ? c.v_scale_slot_stride : c.k_scale_slot_stride;
    float* base = is_v ? c.v_scale + h * c.v_scale_head_stride : c.k_scale + h * c.k_scale_head_stride;
    move_units<float>(kept, a.budget, 1, [&](int i) {
      const int p = a.page_of(i);
      return base + table[p] * page_stride + (i - p * c.page_size) * slot_stride;
    });
  }
}

}  // namespace tris

using namespace tris;

extern "C" int tris_paged_cache_evict(const tris_paged_cache* cache, float* weight_sum, int64_t sum_seq_stride,
                                      int64_t sum_head_stride, int32_t budget, int32_t limit, int32_t sink,
                                      int32_t recent, int32_t* new_lens, int32_t* kept, void* stream) {
  const char* who = "tris_paged_cache_evict";
  if (const int rc = check_paged_cache(who, cache, cache && is_16bit(cache->dtype) ? cache->dtype : TRIS_DTYPE_F16))
    return rc;
  const tris_paged_cache& c = *cache;
  TRIS_REQUIRE(budget >= 1 && limit >= budget, "%s: 1 <= budget <= limit", who);
  TRIS_REQUIRE(sink >= 0 && recent >= 0 && static_cast<int64_t>(sink) + recent <= budget,
               "%s: sink and recent must be within the budget", who);
  if (c.batch == 0) return TRIS_OK;
  TRIS_REQUIRE((weight_sum || c.max_pages == 0) && new_lens && kept, "%s: null pointer", who);
  TRIS_REQUIRE(new_lens != c.seq_lens, "%s: new_lens must not be seq_lens", who);
  TRIS_REQUIRE(cache_rows_apart(c), "%s: cache rows overlap", who);
  TRIS_REQUIRE(cache_scales_apart(c), "%s: cache scales overlap", who);
  TRIS_REQUIRE(sum_rows_apart(c, sum_seq_stride, sum_head_stride), "%s: rows of weight_sum overlap", who);
  const int slices = c.head_dim * (c.dtype == TRIS_DTYPE_E4M3 ? 1 : 2) / kSliceBytes;
  const int parts = 2 * slices + (c.dtype == TRIS_DTYPE_E4M3 ? 3 : 1);
  const int64_t rows = static_cast<int64_t>(c.batch) * c.kv_heads;
  TRIS_REQUIRE(rows * parts < (1LL << 32) / kMoveThreads, "%s: too many rows", who);  // a launch has less than 2^32 threads
  const EvictArgs a{weight_sum, sum_seq_stride, sum_head_stride, budget, limit, sink, recent, new_lens, kept,
                    PageDivision(c.page_size), c};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(evict_select_kernel, dim3(static_cast<unsigned>(rows)), dim3(kSelectThreads), 0, st, a);
  hipLaunchKernelGGL(evict_move_kernel, dim3(static_cast<unsigned>(rows * parts)), dim3(kMoveThreads), 0, st, a, slices,
                     parts);
  return check_launch(who);
}
