// Eviction from the paged cache by accumulated attention weight: which positions stay, and the move of what they hold.
//
// Which: for each (sequence, kv head) the want-th largest weight w* of those between the first `sink` and the last
// `recent` positions, want = budget - sink - recent; above w* all stay, of those equal to it the lowest positions.  w* is
// found digit by digit of a 32-bit key that orders the weights: 11, 11 and 10 bits, each by a histogram in LDS of the keys
// that share the digits before.  The first digit is the sign, the exponent and two bits more, so that weights over many
// powers of two spread over its bins (8-bit digits put two powers of two into one, and the additions wait for each other).
//
// Up to 16384 or 32768 positions one workgroup has a row, its weights in LDS, read once; it lists the positions that
// stay and moves the sums as well, and keys and values too where rows are many or small.  Longer rows are cut into segments
// of a workgroup each, in three launches: histograms of the first digit; the keys in the border's bin, gathered; and, in
// every workgroup alike, the border among those, by which it places its segment.
//
// The choice is bound by latencies and instructions (4225 positions 9.9 us: their way to LDS 1.9, a digit 1.2 to 1.4, the
// classes 1.3, the places 0.7, between launch and end; 131072 positions in segments 4.9 + 6.4 + 9.3), the move by memory:
// each row that changes its place is read and written once.  16 sequences of 8 kv heads with 128 dimensions that go from
// 4225 to 4096 positions (194 MB read, 194 written) 89 us, 4.4 TB/s, of a large copy's 5.15; one of 131072 to 16384 with 4
// kv heads 9.8 + 14.8 us (64 MB); 32 of 1500 to 8192 on e4m3 in one launch with the choice 59 us (237 MB).  Times beside
// the choices below are of whole calls in a graph.
#include "tris_paged.h"

namespace tris {

constexpr int kThreads = 1024;  // of the workgroups of long rows, and of the moves
constexpr int kBlockWaves = kThreads / kWave;
// bits of the digits, first to last, of rows in one workgroup and in segments (whose histograms of the first every workgroup
// of the row reads)
constexpr int kRowBits[3] = {11, 11, 10}, kSegmentBits[3] = {10, 11, 11};
constexpr int kBins = 1 << 11, kFirstBins = 1 << kSegmentBits[0], kFirstShift = 32 - kSegmentBits[0];
constexpr int kMostSegments = 64;  // a lane each
constexpr int kCus = 256, kXcds = 8;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct EvictArgs {
  float* sums;
  int64_t sum_seq, sum_head;
  int32_t budget, limit, sink, recent;
  int32_t* new_lens;
  int32_t* kept;
  PageDivision page_of;
  tris_paged_cache c;
  // of rows in segments
  int32_t segments, segment;  // how many, and positions of one
  int32_t* state;             // [rows][kState]
  int32_t* counts;            // [rows][segments][2]: keys above the bin; keys in it of the segments before
  uint32_t* hist;             // [rows][segments][kFirstBins]
  uint32_t* found;            // [rows][segments * segment]: the keys in the bin, in order
  float* moved;               // [rows][budget]: the sums of what stays
};

// Of a row in segments: whether it is left alone, the border's first digit, how many keys of its bin stay, how many it has.
constexpr int kState = 4, kAlone = 0, kDigit = 1, kWanted = 2, kTotal = 3;

// A weight as an unsigned number of the same order: NaN above all, the zeros equal.
__device__ __forceinline__ uint32_t order_key(float w) {
  const uint32_t u = __float_as_uint(w + 0.0f);  // (-0 + 0 is 0)
  const uint32_t key = u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
  return w != w ? 0xFFFFFFFFu : key;
}

__device__ __forceinline__ int evict_length(const EvictArgs& a, int b) {
  return min(max(a.c.seq_lens[b], 0), cache_positions(a.c));
}

// Whether all pages of a sequence of n > 0 positions are in the pool (for the whole workgroup).
template <int kBlock>
__device__ __forceinline__ bool pages_good(const EvictArgs& a, int b, int n) {
  const int32_t* table = a.c.block_table + b * a.c.table_stride;
  const int last = a.page_of(n - 1);
  bool good = true;
  for (int i = threadIdx.x; i <= last; i += kBlock)
    good = good && static_cast<uint32_t>(table[i]) < static_cast<uint32_t>(a.c.num_pages);
  return __syncthreads_and(good);
}

// The bin, of kCount counted from the largest down, that holds the left-th largest key, how many are above it and in it.
// count(bin): the keys in a bin; a thread asks for kCount / kBlock of them, from kCount - 1 - thread * kCount / kBlock down.
// For the whole workgroup.
template <int kBlock>
struct Pick {
  int bin, above, in;
  int totals[kBlock / kWave];
};
template <int kBlock, int kCount, typename Count>
__device__ __forceinline__ void pick_bin(Count count, int left, Pick<kBlock>* sh) {
  constexpr int kEach = kCount / kBlock;
  const int thread = threadIdx.x, lane = thread % kWave, wave = thread / kWave, high = kCount - 1 - kEach * thread;
  int c[kEach], sum = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) sum += c[i] = count(high - i);
  const int end = wave_incl_sum_i32(sum);
  if (lane == kWave - 1) sh->totals[wave] = end;
  __syncthreads();
  const int total = lane < kBlock / kWave ? sh->totals[lane] : 0, ends = wave_incl_sum_i32(total);
  int before = end - sum + __builtin_amdgcn_readlane(ends - total, wave);
  if (before < left && left <= before + sum) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (before < left && left <= before + c[i]) {
        sh->bin = high - i;
        sh->above = before;
        sh->in = c[i];
      }
      before += c[i];
    }
  }
  __syncthreads();
}

// ------------------------------------------------------------------------------------------------ the move in place

// A row of bytes or one 4-byte number of each position of one kv head: where a position's is.  Positions and pages are
// checked again here, so that tables, lengths or sums that change meanwhile lead nowhere else.
struct Units {
  char* base;
  const int32_t* table;
  int64_t page_bytes;
  int32_t slot_bytes, page_size, num_pages, positions;
  PageDivision page_of;
  __device__ bool valid(int page) const { return static_cast<uint32_t>(page) < static_cast<uint32_t>(num_pages); }
  __device__ char* at(int i, int page) const {
    return base + page * page_bytes + static_cast<int64_t>(i - page_of(i) * page_size) * slot_bytes;
  }
};

// What a move's workgroup of part number `part` has of kv head h's cache: slices of the rows of keys, then of values, then
// the scales.
__device__ __forceinline__ Units part_units(const EvictArgs& a, int b, int h, int part, int slices, int slice_bytes) {
  const tris_paged_cache& c = a.c;
  const int32_t* table = c.block_table + b * c.table_stride;
  if (part < 2 * slices) {
    const bool v = part >= slices;
    const int size = c.dtype == TRIS_DTYPE_E4M3 ? 1 : 2;
    return Units{static_cast<char*>(v ? c.v : c.k) + (v ? c.v_head_stride : c.k_head_stride) * size * h +
                     (v ? part - slices : part) * slice_bytes,
                 table,
                 (v ? c.v_page_stride : c.k_page_stride) * size,
                 static_cast<int32_t>(v ? c.v_slot_stride : c.k_slot_stride) * size,
                 c.page_size,
                 c.num_pages,
                 cache_positions(c),
                 a.page_of};
  }
  const bool v = part > 2 * slices;
  return Units{reinterpret_cast<char*>(v ? c.v_scale : c.k_scale) + (v ? c.v_scale_head_stride : c.k_scale_head_stride) * 4 * h,
               table,
               (v ? c.v_scale_page_stride : c.k_scale_page_stride) * 4,
               static_cast<int32_t>(v ? c.v_scale_slot_stride : c.k_scale_slot_stride) * 4,
               c.page_size,
               c.num_pages,
               cache_positions(c),
               a.page_of};
}

// In place: a workgroup has a slice of every row of one (sequence, kv head), so that no other reads what it writes.  It
// takes the rows in runs from the first place on: a place is never past where its row comes from, so what a run writes no
// later run reads, and its own rows are in registers before any is written.  So a run's rows are asked for before the one
// before it is stored, their pages before that, and the list before that (16 sequences of 4225 190 us one after the other,
// 109 so, both with slices of 64 bytes).  Rows from `end` on are left to the second move.
constexpr int kMoveUnits = 4;

template <typename T, int kBlock>
__device__ __forceinline__ void shift_units(const int32_t* kept, int budget, int end, int lanes, int unit, const Units& u) {
  const int thread = threadIdx.x, rows = kBlock / lanes, first = thread / lanes;
  const int run = rows * kMoveUnits;
  int last = budget;  // no row from here on comes from before `end`
  if (end < INT32_MAX) {
    const int each = (budget + kBlock - 1) / kBlock;
    last = min(budget, each * __syncthreads_count(thread * each < budget && kept[thread * each] < end));
  }
  // of a unit: where its row comes from and goes (its own place: nowhere), their pages, the row
  struct Listed {
    int from[kMoveUnits];
  };
  struct Paged {
    int from[kMoveUnits], from_page[kMoveUnits], to_page[kMoveUnits];
  };
  const auto list = [&](int i0) {
    Listed l;
#pragma unroll
    for (int k = 0; k < kMoveUnits; ++k) {
      const int i = i0 + k * rows + first;
      l.from[k] = i < last ? kept[i] : i;
    }
    return l;
  };
  const auto pages = [&](int i0, const Listed& l) {
    Paged p;
#pragma unroll
    for (int k = 0; k < kMoveUnits; ++k) {
      const int i = i0 + k * rows + first;
      const bool moves = l.from[k] > i && l.from[k] < min(end, u.positions);
      p.from[k] = l.from[k];
      p.from_page[k] = moves ? u.table[u.page_of(l.from[k])] : -1;
      p.to_page[k] = moves ? u.table[u.page_of(i)] : -1;
    }
    return p;
  };
  struct Rows {
    T x[kMoveUnits];
    char* to[kMoveUnits];
  };
  const auto load = [&](int i0, const Paged& p) {
    Rows r;
#pragma unroll
    for (int k = 0; k < kMoveUnits; ++k) {
      const bool moves = u.valid(p.from_page[k]) && u.valid(p.to_page[k]);
      r.x[k] = T{};
      if (moves) r.x[k] = reinterpret_cast<const T*>(u.at(p.from[k], p.from_page[k]))[unit];
      r.to[k] = moves ? u.at(i0 + k * rows + first, p.to_page[k]) : nullptr;
    }
    return r;
  };
  Listed listed = list(run);
  Paged paged = pages(0, list(0));
  Rows now = load(0, paged);
  paged = pages(run, listed);
  listed = list(2 * run);
  for (int i0 = 0; i0 < last; i0 += run) {
    const Paged next = pages(i0 + 2 * run, listed);
    listed = list(i0 + 3 * run);
    Rows ahead = load(i0 + run, paged);
    paged = next;
    // the run's rows have arrived in every wavefront before any stores
#pragma unroll
    for (int k = 0; k < kMoveUnits; ++k) asm volatile("" : "+v"(now.x[k])::"memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int k = 0; k < kMoveUnits; ++k)
      if (now.to[k]) reinterpret_cast<T*>(now.to[k])[unit] = now.x[k];
    now = ahead;
  }
}

// ------------------------------------------------------------------------------------------------ a row in one workgroup

// kMove: the workgroup moves its row's keys and values as well.
template <int kBlock, int kKeys, bool kMove>
__global__ __launch_bounds__(kBlock) void evict_select_kernel(const EvictArgs a) {
  constexpr int kWaves = kBlock / kWave, kCounts = kKeys * kWaves;
  __shared__ float weights[kBlock * kKeys];  // (a position is read by the thread that wrote it)
  __shared__ int hist[kBins];
  __shared__ uint32_t counts[kCounts];
  __shared__ Pick<kBlock> pick;
  const int row = blockIdx.x, b = row / a.c.kv_heads, h = row - b * a.c.kv_heads;
  const int thread = threadIdx.x, lane = thread % kWave, wave = thread / kWave;
  const int n = evict_length(a, b);
  int32_t* kept = a.kept + static_cast<int64_t>(row) * a.budget;
  float* sums = a.sums + b * a.sum_seq + h * a.sum_head;
  bool due = n > a.limit;
  if (due) {
    constexpr int kAtOnce = 8;
#pragma unroll 1
    for (int i0 = thread; i0 < n; i0 += kAtOnce * kBlock) {
      float w[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) w[u] = i0 + u * kBlock < n ? sums[i0 + u * kBlock] : 0.0f;
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) weights[i0 + u * kBlock] = w[u];
    }
    due = pages_good<kBlock>(a, b, n);
  }
  if (h == 0 && thread == 0) a.new_lens[b] = due ? a.budget : a.c.seq_lens[b];
  if (!due) {
    for (uint32_t i = thread; i < static_cast<uint32_t>(a.budget); i += kBlock) kept[i] = -1;  // (a step past 2^31 at most)
    return;
  }
  const int lo = a.sink, hi = n - a.recent, want = a.budget - a.sink - a.recent;
  uint32_t border = 0xFFFFFFFFu;
  int equal = 0;  // of the keys equal to the border, how many stay
  if (want > 0) {
    uint32_t prefix = 0;
    equal = want;
#pragma unroll 1
    for (int shift = 32, bits; shift > 0;) {
      bits = shift > kRowBits[2] ? kRowBits[0] : kRowBits[2];
      shift -= bits;
#pragma unroll
      for (int i = thread; i < kBins; i += kBlock) hist[i] = 0;
      __syncthreads();
      // (64-bit shifts: the first digit has nothing before it)
#pragma unroll 2
      for (int i = thread; i < hi; i += kBlock) {
        const uint32_t key = order_key(weights[i]);
        if (i >= lo && static_cast<uint64_t>(key) >> (shift + bits) == prefix)
          atomicAdd(&hist[key >> shift & ((1u << bits) - 1)], 1);
      }
      __syncthreads();
      pick_bin<kBlock, kBins>([&](int bin) { return hist[bin]; }, equal, &pick);
      prefix = prefix << bits | static_cast<uint32_t>(pick.bin);
      equal -= pick.above;
      border = prefix;
      if (equal == pick.in) {
        // the whole bin stays: the border is the largest key below it (there is one: no key is below 2^22)
        border = (prefix << shift) - 1;
        equal = 0;
        break;
      }
    }
  }
  // Of each 64 positions: how many stay for certain, and (from bit 16 on) how many are equal to the border.
  uint32_t mine = 0;                  // lane j: of the wavefront's 64 from j * kBlock on
  uint32_t sure_bits = 0, tie_bits = 0;  // bit j: of the thread's own
#pragma unroll 1
  for (int j = 0; j * kBlock < n; ++j) {
    const int i = j * kBlock + thread;
    const uint32_t key = order_key(weights[i]);
    const bool middle = i >= lo && i < hi, decides = middle && want > 0;
    const bool sure = decides ? key > border : !middle && i < n, tie = decides && key == border;
    sure_bits |= static_cast<uint32_t>(sure) << j;
    tie_bits |= static_cast<uint32_t>(tie) << j;
    const uint32_t both = __popcll(__ballot(sure)) | __popcll(__ballot(tie)) << 16;
    mine = lane == j ? both : mine;
  }
  if (lane < kKeys) counts[lane * kWaves + wave] = mine;
  __syncthreads();
  if (wave == 0) {  // the numbers before each
    constexpr int kEach = kCounts / kWave;
    uint32_t c[kEach], sum = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) sum += c[i] = counts[lane * kEach + i];
    uint32_t before = static_cast<uint32_t>(wave_incl_sum_i32(static_cast<int>(sum))) - sum;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      counts[lane * kEach + i] = before;
      before += c[i];
    }
  }
  __syncthreads();
  const uint64_t below = (1ull << lane) - 1;
#pragma unroll 1
  for (int j = 0; j * kBlock < n; ++j) {
    const int i = j * kBlock + thread;
    const bool sure = sure_bits >> j & 1, tie = tie_bits >> j & 1;
    const uint32_t before = counts[j * kWaves + wave];
    const int sures = static_cast<int>(before & 0xFFFF) + __popcll(__ballot(sure) & below);
    const int ties = static_cast<int>(before >> 16) + __popcll(__ballot(tie) & below);
    if (sure || (tie && ties < equal)) {
      const int place = sures + min(ties, equal);
      // (outside the budget, on either side, only if the lengths change meanwhile)
      if (static_cast<uint32_t>(place) < static_cast<uint32_t>(a.budget)) {
        kept[place] = i;
        sums[place] = weights[i];  // (the row's weights are all in LDS)
      }
    }
  }
  for (int i = a.budget + thread; i < n; i += kBlock) sums[i] = 0.0f;
  if constexpr (kMove) {
    __syncthreads();
    const bool e4m3 = a.c.dtype == TRIS_DTYPE_E4M3;
    const int lanes = a.c.head_dim * (e4m3 ? 1 : 2) / 16;  // of a row; the values beside the keys
    const bool v = thread % (2 * lanes) >= lanes;
    shift_units<u32x4, kBlock>(kept, a.budget, INT32_MAX, 2 * lanes, thread % lanes, part_units(a, b, h, v, 1, 0));
    if (e4m3) shift_units<uint32_t, kBlock>(kept, a.budget, INT32_MAX, 2, 0, part_units(a, b, h, 2 + thread % 2, 1, 0));
  }
}

// ------------------------------------------------------------------------------------------------ rows in segments

struct Segment {
  int row, s, b, h, n, begin, end;
  __device__ explicit Segment(const EvictArgs& a) {
    row = blockIdx.x / a.segments;
    s = blockIdx.x - row * a.segments;
    b = row / a.c.kv_heads;
    h = row - b * a.c.kv_heads;
    n = evict_length(a, b);
    begin = static_cast<int>(min(static_cast<int64_t>(s) * a.segment, static_cast<int64_t>(n)));
    end = static_cast<int>(min(static_cast<int64_t>(n), static_cast<int64_t>(begin) + a.segment));
  }
  __device__ int64_t index(const EvictArgs& a) const { return static_cast<int64_t>(row) * a.segments + s; }
};

// Four positions of a thread from i0 on, kThreads apart, and their weights.
constexpr int kTileKeys = 4;
constexpr int kTile = kTileKeys * kThreads;

struct Weights {
  float w[kTileKeys];
  __device__ Weights(const EvictArgs& a, const Segment& g, int i0) {
    const float* sums = a.sums + g.b * a.sum_seq + g.h * a.sum_head;
#pragma unroll
    for (int j = 0; j < kTileKeys; ++j) {
      const int i = i0 + j * kThreads + static_cast<int>(threadIdx.x);
      w[j] = i < g.end ? sums[i] : 0.0f;
    }
  }
};

__global__ __launch_bounds__(kThreads) void evict_histogram_kernel(const EvictArgs a) {
  static_assert(kFirstBins == kThreads, "a bin for each thread");
  __shared__ uint32_t hist[kFirstBins];
  const Segment g(a);
  const int thread = threadIdx.x;
  hist[thread] = 0;
  Weights now(a, g, g.begin);
  const bool due = g.n > a.limit && pages_good<kThreads>(a, g.b, g.n);
  if (g.s == 0 && thread == 0) {
    if (g.h == 0) a.new_lens[g.b] = due ? a.budget : a.c.seq_lens[g.b];
    a.state[kState * g.row + kAlone] = !due;
  }
  if (!due) {
    int32_t* kept = a.kept + static_cast<int64_t>(g.row) * a.budget;
    const uint32_t step = a.segments * kThreads;
    for (uint32_t i = g.s * kThreads + thread; i < static_cast<uint32_t>(a.budget); i += step) kept[i] = -1;
    return;
  }
  const int lo = max(g.begin, a.sink), hi = min(g.end, g.n - a.recent);
  for (int i0 = g.begin; i0 < hi; i0 += kTile) {
    if (i0 > g.begin) now = Weights(a, g, i0);
#pragma unroll
    for (int j = 0; j < kTileKeys; ++j) {
      const int i = i0 + j * kThreads + thread;
      if (i >= lo && i < hi) atomicAdd(&hist[order_key(now.w[j]) >> kFirstShift], 1u);
    }
  }
  __syncthreads();
  a.hist[g.index(a) * kFirstBins + thread] = hist[thread];
}

__global__ __launch_bounds__(kThreads) void evict_gather_kernel(const EvictArgs a) {
  __shared__ Pick<kThreads> pick;
  __shared__ int counts[kTileKeys * kBlockWaves];
  __shared__ int above, offset, total;
  const Segment g(a);
  if (a.state[kState * g.row + kAlone]) return;
  const int thread = threadIdx.x, lane = thread % kWave, wave = thread / kWave;
  const int want = a.budget - a.sink - a.recent;
  Weights now(a, g, g.begin);
  // the row's histogram: a bin a thread, from the largest down
  const uint32_t* row_hist = a.hist + static_cast<int64_t>(g.row) * a.segments * kFirstBins;
  const int own = kFirstBins - 1 - thread;
  int count = 0, mine = 0;
#pragma unroll 16
  for (int s = 0; s < a.segments; ++s) {
    const int c = row_hist[static_cast<int64_t>(s) * kFirstBins + own];
    count += c;
    mine = s == g.s ? c : mine;
  }
  if (thread == 0) {
    pick.bin = kFirstBins;  // where nothing is wanted: no key is above it, none in it
    pick.above = above = 0;
  }
  __syncthreads();
  if (want > 0) pick_bin<kThreads, kFirstBins>([&](int) { return count; }, want, &pick);
  const int bin = pick.bin;
  mine = wave_incl_sum_i32(own > bin ? mine : 0);
  if (lane == kWave - 1 && mine) atomicAdd(&above, mine);
  // the keys in the bin, of the segments before and of all
  if (wave == 0) {
    const int in = lane < a.segments && bin < kFirstBins ? row_hist[static_cast<int64_t>(lane) * kFirstBins + bin] : 0;
    const int end = wave_incl_sum_i32(in);
    if (lane == g.s) offset = end - in;
    if (lane == kWave - 1) total = end;
  }
  __syncthreads();
  if (thread == 0) {
    a.counts[2 * g.index(a)] = above;
    a.counts[2 * g.index(a) + 1] = offset;
    if (g.s == 0) {
      a.state[kState * g.row + kDigit] = bin;
      a.state[kState * g.row + kWanted] = want - pick.above;
      a.state[kState * g.row + kTotal] = total;
    }
  }
  // its keys, in order
  uint32_t* found = a.found + static_cast<int64_t>(g.row) * a.segments * a.segment;
  const int lo = max(g.begin, a.sink), hi = min(g.end, g.n - a.recent);
  int placed = offset;
  for (int i0 = g.begin; i0 < hi; i0 += kTile) {
    if (i0 > g.begin) now = Weights(a, g, i0);
    uint64_t in[kTileKeys];
#pragma unroll
    for (int j = 0; j < kTileKeys; ++j) {
      const int i = i0 + j * kThreads + thread;
      in[j] = __ballot(i >= lo && i < hi && static_cast<int>(order_key(now.w[j]) >> kFirstShift) == bin);
      if (lane == 0) counts[j * kBlockWaves + wave] = __popcll(in[j]);
    }
    __syncthreads();
    const int c = counts[lane], end = wave_incl_sum_i32(c);  // (each wavefront: the tile's 64 counts)
#pragma unroll
    for (int j = 0; j < kTileKeys; ++j) {
      const int before = __shfl(end - c, j * kBlockWaves + wave);
      if (in[j] >> lane & 1) found[placed + before + __popcll(in[j] & ((1ull << lane) - 1))] = order_key(now.w[j]);
    }
    placed += __builtin_amdgcn_readlane(end, kWave - 1);
    __syncthreads();
  }
}

__global__ __launch_bounds__(kThreads) void evict_place_kernel(const EvictArgs a) {
  __shared__ int hist[kBins];
  __shared__ Pick<kThreads> pick;
  __shared__ int before[2];      // of the segments before: positions that stay for certain, keys equal to the border
  __shared__ int counts[kTileKeys * kBlockWaves];
  const Segment g(a);
  const int32_t* state = a.state + kState * g.row;
  if (state[kAlone]) return;
  const int thread = threadIdx.x, lane = thread % kWave, wave = thread / kWave;
  const int first = state[kDigit], total = state[kTotal], lo = a.sink, hi = g.n - a.recent;
  Weights now(a, g, g.begin);
  const int2* row_counts = reinterpret_cast<const int2*>(a.counts) + static_cast<int64_t>(g.row) * a.segments;
  const int offset = row_counts[g.s].y;
  // every key of the row's bin, the first of a thread's in registers
  const uint32_t* found = a.found + static_cast<int64_t>(g.row) * a.segments * a.segment;
  uint32_t key[kTileKeys];
#pragma unroll
  for (int j = 0; j < kTileKeys; ++j) key[j] = j * kThreads + thread < total ? found[j * kThreads + thread] : 0u;
  const auto each = [&](auto&& f) {
#pragma unroll
    for (int j = 0; j < kTileKeys; ++j)
      if (j * kThreads + thread < total) f(j * kThreads + thread, key[j]);
#pragma unroll 4
    for (int i = kTile + thread; i < total; i += kThreads) f(i, found[i]);
  };
  if (thread < 2) before[thread] = 0;
  __syncthreads();
  if (thread < g.s) {
    const int begin = static_cast<int>(min(static_cast<int64_t>(thread) * a.segment, static_cast<int64_t>(g.n)));
    const int end = static_cast<int>(min(static_cast<int64_t>(g.n), static_cast<int64_t>(begin) + a.segment));
    // (and the first and last positions, which are held)
    atomicAdd(&before[0], row_counts[thread].x + max(0, min(end, lo) - begin) + max(0, end - max(begin, hi)));
  }
  const bool some = first < kFirstBins;
  uint32_t border = 0xFFFFFFFFu;
  int equal = 0;
  if (some) {
    border = static_cast<uint32_t>(first);
    equal = state[kWanted];
#pragma unroll
    for (int digit = 1; digit < 3; ++digit) {
      constexpr int kLast = kSegmentBits[2];
      const int shift = digit == 1 ? kLast : 0, bits = kSegmentBits[digit];
      hist[thread] = hist[thread + kThreads] = 0;
      __syncthreads();
      each([&](int, uint32_t k) {
        if (k >> (shift + bits) == border) atomicAdd(&hist[k >> shift & ((1 << bits) - 1)], 1);
      });
      __syncthreads();
      pick_bin<kThreads, kBins>([&](int bin) { return hist[bin]; }, equal, &pick);
      border = border << bits | static_cast<uint32_t>(pick.bin);
      equal -= pick.above;
      if (digit == 1 && equal == pick.in) {  // (as above)
        border = (border << shift) - 1;
        equal = 0;
        break;
      }
    }
    int sure = 0, ties = 0;
    each([&](int i, uint32_t k) {
      sure += i < offset && k > border;
      ties += i < offset && k == border;
    });
    sure = wave_incl_sum_i32(sure);
    ties = wave_incl_sum_i32(ties);
    if (lane == kWave - 1) {
      atomicAdd(&before[0], sure);
      atomicAdd(&before[1], ties);
    }
  }
  __syncthreads();
  int sures = before[0], tied = before[1];
  int32_t* kept = a.kept + static_cast<int64_t>(g.row) * a.budget;
  float* moved = a.moved + static_cast<int64_t>(g.row) * a.budget;
  float* sums = a.sums + g.b * a.sum_seq + g.h * a.sum_head;
  for (int i0 = g.begin; i0 < g.end; i0 += kTile) {
    if (i0 > g.begin) now = Weights(a, g, i0);
    uint64_t sure[kTileKeys], tie[kTileKeys];
#pragma unroll
    for (int j = 0; j < kTileKeys; ++j) {
      const int i = i0 + j * kThreads + thread;
      const uint32_t k = order_key(now.w[j]);
      const bool middle = some && i >= lo && i < hi;
      sure[j] = __ballot(i < g.end && (i < lo || i >= hi || (middle && k > border)));
      tie[j] = __ballot(i < g.end && middle && k == border);
      if (lane == 0) counts[j * kBlockWaves + wave] = __popcll(sure[j]) | __popcll(tie[j]) << 16;
    }
    __syncthreads();
    const int c = counts[lane], end = wave_incl_sum_i32(c);
    const uint64_t below = (1ull << lane) - 1;
#pragma unroll
    for (int j = 0; j < kTileKeys; ++j) {
      const int past = __shfl(end - c, j * kBlockWaves + wave);
      const int t = tied + (past >> 16) + __popcll(tie[j] & below);
      const int place = sures + (past & 0xFFFF) + __popcll(sure[j] & below) + min(t, equal);
      const bool stays = (sure[j] >> lane & 1) || ((tie[j] >> lane & 1) && t < equal);
      // (outside the budget, on either side, only if the sums change meanwhile)
      if (stays && static_cast<uint32_t>(place) < static_cast<uint32_t>(a.budget)) {
        kept[place] = i0 + j * kThreads + thread;
        moved[place] = now.w[j];
      }
    }
    const int all = __builtin_amdgcn_readlane(end, kWave - 1);
    sures += all & 0xFFFF;
    tied += all >> 16;
    // (no other workgroup reads this segment's sums, and what stays is in `moved`)
#pragma unroll
    for (int j = 0; j < kTileKeys; ++j) {
      const int i = i0 + j * kThreads + thread;
      if (i >= a.budget && i < g.end) sums[i] = 0.0f;
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------------ the moves

// parts: of a row: slices of keys, then of values, the scales, and where the row is in segments the sums.
__global__ __launch_bounds__(kThreads) void evict_shift_kernel(const EvictArgs a, int slices, int slice_bytes, int parts,
                                                               int end) {
  // a row's parts on one XCD, whose cache then has a line for both of its slices
  const int group = blockIdx.x / (kXcds * parts), in = blockIdx.x - group * (kXcds * parts);
  const int row = group * kXcds + in % kXcds, part = in / kXcds;
  if (row >= a.c.batch * a.c.kv_heads) return;
  const int b = row / a.c.kv_heads, h = row - b * a.c.kv_heads;
  const int32_t* kept = a.kept + static_cast<int64_t>(row) * a.budget;
  if (kept[0] < 0) return;
  const int thread = threadIdx.x;
  if (a.segments > 0 && part == parts - 1) {
    float* sums = a.sums + b * a.sum_seq + h * a.sum_head;
    const float* moved = a.moved + static_cast<int64_t>(row) * a.budget;
    const int n = min(a.budget, evict_length(a, b));
#pragma unroll 4
    for (int i = thread; i < n; i += kThreads) sums[i] = moved[i];
    return;
  }
  const Units u = part_units(a, b, h, part, slices, slice_bytes);
  const int lanes = slice_bytes / 16;
  if (part < 2 * slices) shift_units<u32x4, kThreads>(kept, a.budget, end, lanes, thread % lanes, u);
  else shift_units<uint32_t, kThreads>(kept, a.budget, end, 1, 0, u);
}

// From positions past the budget, which no move writes: after the first move in any order, by any number of workgroups.
constexpr int kFetchUnits = 2;

template <typename T>
__device__ __forceinline__ void fetch_units(const int32_t* kept, int budget, int lanes, int i0, int step, const Units& u) {
  const int unit = threadIdx.x % lanes;
  for (int i = i0; i < budget; i += step * kFetchUnits) {
    T x[kFetchUnits] = {};
    char* to[kFetchUnits];
    int from[kFetchUnits], from_page[kFetchUnits], to_page[kFetchUnits];
#pragma unroll
    for (int k = 0; k < kFetchUnits; ++k) from[k] = i + k * step < budget ? kept[i + k * step] : -1;
#pragma unroll
    for (int k = 0; k < kFetchUnits; ++k) {
      const bool moves = from[k] >= budget && from[k] < u.positions;
      from_page[k] = moves ? u.table[u.page_of(from[k])] : -1;
      to_page[k] = moves ? u.table[u.page_of(i + k * step)] : -1;
    }
#pragma unroll
    for (int k = 0; k < kFetchUnits; ++k) {
      const bool moves = u.valid(from_page[k]) && u.valid(to_page[k]);
      if (moves) x[k] = reinterpret_cast<const T*>(u.at(from[k], from_page[k]))[unit];
      to[k] = moves ? u.at(i + k * step, to_page[k]) : nullptr;
    }
#pragma unroll
    for (int k = 0; k < kFetchUnits; ++k)
      if (to[k]) reinterpret_cast<T*>(to[k])[unit] = x[k];
  }
}

constexpr int kFetchThreads = 256;
constexpr int kFetchBlocks = 2048;  // of keys and values, at least, where there is work for them

__global__ __launch_bounds__(kFetchThreads, 8) void evict_fetch_kernel(const EvictArgs a, int row_bytes, int parts,
                                                                       int splits) {
  const int split = blockIdx.x % splits, unit = blockIdx.x / splits, row = unit / parts, part = unit - row * parts;
  const int b = row / a.c.kv_heads, h = row - b * a.c.kv_heads;
  const int32_t* kept = a.kept + static_cast<int64_t>(row) * a.budget;
  if (kept[0] < 0) return;
  const Units u = part_units(a, b, h, part, 1, row_bytes);
  const int lanes = part < 2 ? row_bytes / 16 : 1, rows = kFetchThreads / lanes;
  const int i0 = split * rows + static_cast<int>(threadIdx.x) / lanes, step = splits * rows;
  if (part < 2) fetch_units<u32x4>(kept, a.budget, lanes, i0, step, u);
  else fetch_units<uint32_t>(kept, a.budget, lanes, i0, step, u);
}

// A row's workgroup has 1024 threads, or 256 where the table is so narrow (256 / 1024: 4 rows of 900 positions 11.7 / 10.4
// us, 320 rows 13.6 / 18.3, of 3000 positions 19.7 / 22.4).
constexpr int kShort = 256, kShortManyRows = 16 * 256;

template <bool kMove>
static void select_launch(const EvictArgs& a, int64_t rows, int64_t positions, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(rows));
  if (positions <= (rows > kCus ? kShortManyRows : kShort))
    hipLaunchKernelGGL((evict_select_kernel<256, 16, kMove>), grid, dim3(256), 0, st, a);
  else if (positions <= 16 * kThreads)
    hipLaunchKernelGGL((evict_select_kernel<kThreads, 16, kMove>), grid, dim3(kThreads), 0, st, a);
  else
    hipLaunchKernelGGL((evict_select_kernel<kThreads, 32, kMove>), grid, dim3(kThreads), 0, st, a);
}

// Slices of 128 bytes from as many workgroups on, else of 64 (the call in a graph, 128 / 64: 64 workgroups of 128 bytes 29.9
// / 23.9 us, 128 33.3 / 29.9, 184 68.0 / 75.3, 512 101.9 / 107.7).
constexpr int kWideSlices = 160;
// The selecting workgroups move what their rows keep, in one launch, where that is up to so many bytes of a row, and, up to
// four times as many or one workgroup a CU, from so many rows on (together / in two launches: 8 rows of 32, 128 and 256
// positions of 512 bytes 8.9 / 10.9, 11.7 / 10.9, 16.1 / 11.7 us in a graph, and a launch less for the host; 192 rows of
// 512 and 2048 23.4 / 32.3, 78 / 85; 320 rows of 512, 1024 and 2048 40 / 44, 86 / 84, 155 / 138).
constexpr int64_t kSmallMove = 64 << 10;
constexpr int kManyRows = 160;
// In a decode loop a sequence is due in one of limit - budget + 1 steps, and in the others a launch less is what counts: so
// they move too where all sequences' moves come to so many bytes of a row a step (one sequence of 8 heads, 2048 positions of
// 512 bytes, limit 2176: 3.9 / 5.5 us with nothing due, 40 / 20 when it is).  A caller who makes the call only when it is due
// gets the second by giving the budget as the limit.
constexpr int64_t kRareMove = 16 << 10;
// Budgets past which the rows from past the budget are moved by a launch of their own, where slices are few and the table has
// twice as many positions (with it / without: 4 rows of 8192 of 65536 positions 35.4 / 42.5 us, 16 rows 56.8 / 67.7; 32 rows of
// 8192 of 32768, which are too many slices, 102.5 / 96.1).  4096 itself is left out, where it goes either way (of 32768, 4 rows
// 43.5 / 46.1, 16 rows 53.5 / 51.1).
constexpr int kFarBudget = 4096;

struct EvictSpace {
  int64_t counts, hist, found, moved, bytes;
  int segments, segment;
};

// Positions of a table up to which a row is one workgroup's: more where rows are many (in segments / in one workgroup: 4 rows
// of 12000 positions 25.7 / 23.8 us, 20000 26.3 / 29.0; 32 rows of 20000 32.0 / 36.0; 128 rows of 32000 93 / 83).
constexpr int kFewRows = 64;
static int64_t one_workgroup(int64_t rows) { return (rows <= kFewRows ? 16 : 32) * kThreads; }

static EvictSpace evict_space(int64_t rows, int64_t positions, int64_t budget) {
  EvictSpace s{};
  if (positions <= one_workgroup(rows)) return s;
  const auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
  s.segments = static_cast<int>(std::min<int64_t>(kMostSegments, (positions + kTile - 1) / kTile));
  const int64_t each = (positions + s.segments - 1) / s.segments;
  s.segment = static_cast<int>((each + kTile - 1) / kTile * kTile);
  s.counts = up(rows * kState * 4);
  s.hist = s.counts + up(rows * 2LL * s.segments * 4);
  s.found = s.hist + rows * s.segments * kFirstBins * 4;
  s.moved = s.found + rows * s.segments * s.segment * 4;
  s.bytes = s.moved + (budget < positions ? rows * budget * 4 : 0);  // (no sequence is due from there on)
  return s;
}

}  // namespace tris

using namespace tris;

extern "C" int64_t tris_paged_cache_evict_workspace_bytes(int32_t batch, int32_t kv_heads, int32_t max_pages,
                                                          int32_t page_size, int32_t budget) {
  if (batch < 1 || kv_heads < 1 || max_pages < 0 || page_size < 1 || budget < 1) return 0;
  if (static_cast<int64_t>(batch) * kv_heads >= (1LL << 32) / kThreads) return 0;  // refused
  return evict_space(static_cast<int64_t>(batch) * kv_heads, static_cast<int64_t>(max_pages) * page_size, budget).bytes;
}

extern "C" int tris_paged_cache_evict(const tris_paged_cache* cache, float* weight_sum, int64_t sum_seq_stride,
                                      int64_t sum_head_stride, int32_t budget, int32_t limit, int32_t sink,
                                      int32_t recent, int32_t* new_lens, int32_t* kept, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
  const char* who = "tris_paged_cache_evict";
  if (const int rc = check_paged_cache(who, cache, cache && is_16bit(cache->dtype) ? cache->dtype : TRIS_DTYPE_F16))
    return rc;
  const tris_paged_cache& c = *cache;
  TRIS_REQUIRE(budget >= 1 && limit >= budget, "%s: 1 <= budget <= limit", who);
  TRIS_REQUIRE(sink >= 0 && recent >= 0 && static_cast<int64_t>(sink) + recent <= budget,
               "%s: sink and recent must be within the budget", who);
  if (c.batch == 0) return TRIS_OK;
  TRIS_REQUIRE((weight_sum || c.max_pages == 0) && new_lens && kept, "%s: null pointer", who);
  TRIS_REQUIRE(cache_rows_apart(c), "%s: cache rows overlap", who);
  TRIS_REQUIRE(cache_scales_apart(c), "%s: cache scales overlap", who);
  TRIS_REQUIRE(sum_rows_apart(c, sum_seq_stride, sum_head_stride), "%s: rows of weight_sum overlap", who);
  const int64_t rows = static_cast<int64_t>(c.batch) * c.kv_heads, positions = cache_positions(c);
  const bool e4m3 = c.dtype == TRIS_DTYPE_E4M3;
  const int row_bytes = c.head_dim * (e4m3 ? 1 : 2);
  const EvictSpace s = evict_space(rows, positions, budget);
  const int64_t row_move = static_cast<int64_t>(budget) * row_bytes * 2;
  const bool small = row_move <= kSmallMove ||
                     static_cast<__int128>(row_move) * c.batch <= kRareMove * (static_cast<__int128>(limit) - budget + 1);
  const bool together =
      s.segments == 0 && (small || (rows >= kManyRows && (rows <= kCus || row_move <= 4 * kSmallMove)));
  const int slice_bytes = row_bytes >= 128 && rows * 2 * (row_bytes / 128) >= kWideSlices ? 128 : 64;
  const int slices = row_bytes / slice_bytes, parts = 2 * slices + (e4m3 ? 2 : 0) + (s.segments ? 1 : 0);
  const bool far = positions >= 2LL * budget && rows * 2 * slices <= kCus / 2 && budget > kFarBudget;
  const int fetch_parts = e4m3 ? 4 : 2;
  const int splits = static_cast<int>(std::min<int64_t>(256, std::max<int64_t>(1, kFetchBlocks / (rows * 2))));
  // a launch has less than 2^32 threads
  TRIS_REQUIRE((rows + kXcds) * std::max(parts, s.segments) < (1LL << 32) / kThreads &&
                   rows * fetch_parts * splits < (1LL << 32) / kFetchThreads,
               "%s: too many rows", who);
  // (the lengths are read after the first new ones, and the first of kept's places, are written)
  const auto over = [](const int32_t* x, int64_t n, const int32_t* y, int64_t m) {
    const auto x0 = reinterpret_cast<uintptr_t>(x), y0 = reinterpret_cast<uintptr_t>(y);
    return x0 < y0 ? (y0 - x0) / 4 < static_cast<uint64_t>(n) : (x0 - y0) / 4 < static_cast<uint64_t>(m);
  };
  TRIS_REQUIRE(!over(new_lens, c.batch, c.seq_lens, c.batch), "%s: new_lens must not overlap seq_lens", who);
  TRIS_REQUIRE(s.bytes == 0 || (workspace && aligned16(workspace) && workspace_bytes >= s.bytes),
               "%s: workspace of %lld bytes needed", who, static_cast<long long>(s.bytes));
  TRIS_REQUIRE(keys_and_values_apart(c), "%s: keys and values must not share memory", who);
  TRIS_REQUIRE(!over(kept, rows * budget, c.seq_lens, c.batch) && !over(kept, rows * budget, new_lens, c.batch),
               "%s: kept must not overlap the lengths", who);
  EvictArgs a{weight_sum, sum_seq_stride, sum_head_stride, budget, limit, sink, recent, new_lens, kept,
              PageDivision(c.page_size), c, s.segments, s.segment, nullptr, nullptr, nullptr, nullptr, nullptr};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (together) {
    select_launch<true>(a, rows, positions, st);
    return check_launch(who);
  }
  if (s.segments == 0) {
    select_launch<false>(a, rows, positions, st);
  } else {
    char* at = static_cast<char*>(workspace);
    a.state = reinterpret_cast<int32_t*>(at);
    a.counts = reinterpret_cast<int32_t*>(at + s.counts);
    a.hist = reinterpret_cast<uint32_t*>(at + s.hist);
    a.found = reinterpret_cast<uint32_t*>(at + s.found);
    a.moved = reinterpret_cast<float*>(at + s.moved);
    const dim3 grid(static_cast<unsigned>(rows * s.segments)), block(kThreads);
    hipLaunchKernelGGL(evict_histogram_kernel, grid, block, 0, st, a);
    hipLaunchKernelGGL(evict_gather_kernel, grid, block, 0, st, a);
    hipLaunchKernelGGL(evict_place_kernel, grid, block, 0, st, a);
  }
  const int64_t shift_blocks = (rows + kXcds - 1) / kXcds * kXcds * parts;
  hipLaunchKernelGGL(evict_shift_kernel, dim3(static_cast<unsigned>(shift_blocks)), dim3(kThreads), 0, st, a, slices,
                     slice_bytes, parts, far ? budget : INT32_MAX);
  if (far)
    hipLaunchKernelGGL(evict_fetch_kernel, dim3(static_cast<unsigned>(rows * fetch_parts * splits)), dim3(kFetchThreads), 0,
                       st, a, row_bytes, fetch_parts, splits);
  return check_launch(who);
}
