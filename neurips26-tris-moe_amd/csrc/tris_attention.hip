// Attention of one new token a sequence over the paged cache.
//
//   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  s_j = scale * q . k_j,  m = max_j s_j
//
// One pass over the keys with the running maximum and sum.  A wavefront takes tiles of 32 keys for up to 16 query
// heads of one kv head, so that each key and value is read once for all of them, and both products run on the matrix
// cores straight from registers:
//   S^T [keys x heads] = K Q^T    two 16x16x32 products a 32-wide slice of head_dim.  A lane's K operand is a run of
//                                 one key's row, its result four keys of one head: lane l has head l % 16 and, of
//                                 each 16 keys, those of its group g = l / 16: 4 g .. 4 g + 3.
//   O^T [dim x heads]  = V^T P^T  the eight probabilities that a lane then holds are the eight that its group has to
//                                 supply as the right operand, if the sum runs over the keys in that order.  The left
//                                 operand wants eight keys of one dimension in a lane; it loads eight keys' rows, a
//                                 run of eight dimensions each, and turns that 8 x 8 block with one v_perm_b32 a word:
//                                 product m of eight takes the m-th dimension of every lane's run.
// No operand but the query at 256 dimensions goes through LDS, the statistics of a head stay in its lanes, and rescaling
// is a product in a lane.
//
// The work is split over the length: the tiles of all sequences and head groups form one line, and each workgroup takes
// an equal stretch of it, so that a long sequence beside short ones is shared by the whole GPU and all workgroups end
// together.  Every wavefront derives the same line from seq_lens, so the launch needs no lengths on the host.  (Where the
// block table is narrow there is no line: each workgroup has a (sequence, head group), in one launch.)
//
// Bound by memory: a (key, kv head) is 4 head_dim bytes in 16 bits and 4 flops a byte for each query head of the group.
// One MI355X reads 6.2 TB/s; 131072 tokens with 4 kv heads of 128 (268 MB) take 45.5 + 4.7 us, 64 sequences of 4000 to
// 8192 tokens on an e4m3 cache (792 MB) 137 + 5.2, 32 of 300 to 6000 in a window of 4096 with 16 kv heads (473 MB) 78 +
// 4.7. Below some 50 MB the way to the first rows (length, page, row: three memory latencies) and the second launch
// bound it: 1000 tokens, 8 kv heads (4 MB) 6.6 + 3.3 us.  More than 16 query heads of a kv head read its rows once for
// each 16: 16 sequences of 32768 with one kv head 56 us for 16 heads, 94 for 20.  A (sequence, head group) that one
// workgroup has whole is written at once; the pieces of one that several share leave fp32 sums in the workspace, and a
// second launch joins them.
//
// The keys' weights (weight_sum[kv head][j] += sum_h exp(s_hj - m_h) / l_h, over the kv head's query heads) need every
// head's m and l before the first of them is known, so the first launch leaves the scaled scores, 4 bytes for each query
// head and key, and the second, beside the join, takes the weights from them: 8 group bytes a key and kv head more than
// 4 head_dim, and 8 for the sum.  What they cost over the call without them: 131072 tokens with 4 kv heads of 8 query heads
// 51 -> 69 us, 64 sequences on e4m3 of 4 query heads a kv head 137 -> 196, 16 ragged 23 -> 29, 1000 tokens 8.8 -> 10.2.  The
// scores' way to memory is most of it: 47 MB of stores cost the second of these 44 us beside its 5.9 TB/s of loads, 1 TB/s
// (a large copy writes at 2.6), in stretches of 64 bytes to 4 KB, cached or written through alike, and nothing where they
// fall on lines that stay in the L2.  Reading the keys again instead would take 23 and 67 us.
//
// Times beside the choices below are of whole calls, kernels and join, in a graph over three states: "128k" and the
// others are the calls named here, "ragged" is 16 sequences of 20 to 8000 tokens on fp16, "wide" 8 of 1000 to 16000 with
// 256 dimensions and pages of 20.
#include <algorithm>

#include "tris_paged.h"

namespace tris {

constexpr int kTileKeys = 32;
constexpr int kWaves = 4;          // wavefronts of a workgroup, taking its tiles in turn
constexpr int kHeadTile = 16;      // query heads of a workgroup
constexpr int kCus = 256;
// Wavefronts a SIMD, and so workgroups a CU, that a head dimension's registers leave room for; a grid of as many runs in
// one go (half as many / as many / twice: 128k 56.3 / 50.9 / 53.6 us, 64 on e4m3 163 / 138 / 142, windowed 99 / 83 / 83,
// ragged 26.5 / 24.2 / 28.2, wide 29.3 / 30.0 / 40.2).
__host__ __device__ constexpr int resident(int head_dim) { return head_dim == 64 ? 4 : head_dim == 128 ? 3 : 2; }
// Cache policy of the rows, which are read once: non-temporal (cached / not: 128k 57.2 / 50.9 us, windowed 92.9 / 83.8, 64
// on e4m3 152 / 138, ragged 23.6 / 24.2).  Where each lane has its row's address, a key row's quarters come by different
// instructions and may lie across lines: there the keys are cached (wide: 30.0, not cached 33.6), the values not (30.1).
constexpr int kLoadOnce = 2;

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

struct AttentionArgs {
  const uint16_t* q;
  uint16_t* out;
  int64_t q_seq, q_head, out_seq, out_head;
  float scale_log2;                  // scale * log2(e): the softmax runs on powers of two
  int32_t window, q_heads, group, head_tiles, tile_heads, workgroups;
  PageDivision page_of;
  int2* owners;                      // [batch][kv_heads * head_tiles]: the first and the last workgroup with a piece of it
  float2* part_ml;                   // [2 * workgroups][tile_heads]: maximum and sum of a piece
  float* part_o;                     // the same rows of head_dim sums
  tris_paged_cache c;
  // of the calls that sum the weights
  float* scores;                     // scale_log2 * q . k, see score_block
  int64_t score_row;                 // keys of a (sequence, query head) there
  float2* whole_ml;                  // [batch][q_heads]: maximum and sum of what one workgroup had whole
  float* weight_sum;
  int64_t sum_seq, sum_head;
  int32_t sums4;                     // the sums' rows can be read four at a time
};

// Whether a workgroup of the attention adds the weights of what it has itself: it has a kv head's keys and query heads
// whole, so that there is no second launch (128 tokens 7.3 us, 9.0 with one; 64 of 100 to 500 21.3, 23.6).
__host__ __device__ inline bool own_weights(const AttentionArgs& a) { return a.owners == nullptr && a.head_tiles == 1; }

// a value that every lane holds alike, moved to a scalar register
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
// A load from global memory (not a generic one, which would count as an LDS access too).  kOnce: of what is not read
// again.
template <typename T, bool kOnce>
__device__ __forceinline__ T load_global(const char* base, uint32_t offset) {
  typedef const __attribute__((address_space(1))) char* Base;
  typedef const __attribute__((address_space(1))) T* Typed;
  if constexpr (kOnce) return __builtin_nontemporal_load((Typed)((Base)base + offset));
  else return *(Typed)((Base)base + offset);
}

// a sequence's token attends to the positions [range_begin, sequence_length)
__device__ __forceinline__ int sequence_length(const AttentionArgs& a, int b) {
  return b < a.c.batch ? min(max(a.c.seq_lens[b], 0), cache_positions(a.c)) : 0;
}
__device__ __forceinline__ int range_begin(const AttentionArgs& a, int n) {
  return a.window > 0 ? max(0, n - a.window) : 0;
}
// A sequence's tiles, an idle one's too: one, without keys, so that some workgroup writes its zeros.
__device__ __forceinline__ int range_tiles(int n, int first) {
  return n > first ? (n + kTileKeys - 1) / kTileKeys - first / kTileKeys : 1;
}

// The line: sequence by sequence, in each its head groups one after the other, in each its tiles and then kPieceCost
// places for what a piece costs whatever its length (its query, the first rows' way from memory, the sums' way out), so
// that a stretch of short sequences is a short one.  Of `total` places workgroup w of `shares` has
// [start(w), start(w + 1)), equal to within one.
// (0, 2, 4, 8, 12 places: ragged 38.1, 26.5, 24.2, 24.8, 25.8 us, wide 35.1, 31.3, 30.0, 29.3, 29.3, windowed 81 to 86
// without an order; one or 64 long ones do not care.)
constexpr int kPieceCost = 4;

typedef const __attribute__((address_space(4))) AttentionArgs* KernelArgs;

struct Line {
  int shares, each, more;
  Line() = default;
  __device__ Line(int total, int workgroups) {
    shares = min(workgroups, (total + kWaves - 1) / kWaves);  // no fewer than one tile for a wavefront
    each = total / shares;
    more = total - each * shares;
  }
  __device__ int start(int w) const { return w * each + min(w, more); }
  __device__ int owner(int x) const {
    return x < more * (each + 1) ? x / (each + 1) : more + (x - more * (each + 1)) / each;
  }
};

// The places and lengths of 64 sequences from b0, one a lane.
__device__ __forceinline__ int places_of(const AttentionArgs& a, int b0, int head_groups, int* n) {
  const int b = b0 + static_cast<int>(threadIdx.x) % kWave;
  *n = sequence_length(a, b);
  return b < a.c.batch ? (range_tiles(*n, range_begin(a, *n)) + kPieceCost) * head_groups : 0;
}

// A workgroup's part of the line, [at, stop), and the sequence where it begins: its number, length and first place.
struct Stretch {
  Line line;
  int at, stop, begin, b, n;
};

__device__ __forceinline__ bool line_stretch(const AttentionArgs& a, int head_groups, int w, Stretch* s) {
  int length0;
  const int places0 = places_of(a, 0, head_groups, &length0), end0 = wave_incl_sum_i32(places0);
  int total = __builtin_amdgcn_readlane(end0, kWave - 1);
  for (int b0 = kWave; b0 < a.c.batch; b0 += kWave) {
    int length;
    total += __builtin_amdgcn_readlane(wave_incl_sum_i32(places_of(a, b0, head_groups, &length)), kWave - 1);
  }
  s->line = Line(total, a.workgroups);
  if (w >= s->line.shares) return false;
  s->at = s->line.start(w);
  s->stop = s->line.start(w + 1);
  for (int b0 = 0, places = places0, end = end0, length = length0;;) {
    const uint64_t past = __ballot(s->at < end);
    if (past) {
      const int l = __builtin_ctzll(past);
      s->begin = __builtin_amdgcn_readlane(end - places, l);
      s->b = b0 + l;
      s->n = __builtin_amdgcn_readlane(length, l);
      return true;
    }
    const int before = __builtin_amdgcn_readlane(end, kWave - 1);
    b0 += kWave;
    if (b0 >= a.c.batch) return false;
    places = places_of(a, b0, head_groups, &length);
    end = before + wave_incl_sum_i32(places);
  }
}

// Without a line: workgroup w has one (sequence, head group), all of it.
__device__ __forceinline__ bool own_stretch(const AttentionArgs& a, int head_groups, int w, Stretch* s) {
  s->b = w / head_groups;
  s->n = uniform(sequence_length(a, s->b));
  const int tiles = range_tiles(s->n, range_begin(a, s->n));
  s->begin = 0;
  s->at = (w - s->b * head_groups) * (tiles + kPieceCost);
  s->stop = s->at + tiles;
  return true;
}

template <bool kBf16>
__device__ __forceinline__ f32x4 mfma(u32x4 x, u32x4 y, f32x4 c) {
  if constexpr (kBf16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, y), c, 0, 0, 0);
}

// two e4m3 values (the low or the high half of a word) as 16-bit values, exactly
template <bool kBf16, bool kHigh>
__device__ __forceinline__ uint32_t from_e4m3(uint32_t w) {
  if constexpr (kBf16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, kHigh));
  else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, kHigh));
}

// a maximum or sum over the four groups of 16 lanes
template <typename Op>
__device__ __forceinline__ float across_groups(float v, Op op) {
  const uint32_t u = __float_as_uint(v);
  const auto x = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  v = op(__uint_as_float(x[0]), __uint_as_float(x[1]));
  const uint32_t w = __float_as_uint(v);
  const auto y = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return op(__uint_as_float(y[0]), __uint_as_float(y[1]));
}

// A piece: the tiles [t0, t1) of sequence b (n positions, from `first` on) and head group hg, at place `at` of the line;
// whole: all the tiles there are; else `slot` takes its sums.
struct Piece {
  int b, n, first, hg, t0, t1, at, slot;
  bool whole;
};

constexpr bool query_in_lds(int head_dim) { return head_dim == 256; }

// element i of a row of 16-bit or e4m3 values
template <bool kBf16, bool kE4m3>
__device__ __forceinline__ float element(const void* rows, int64_t i) {
  if constexpr (kE4m3) return __builtin_amdgcn_cvt_f32_fp8(static_cast<const uint8_t*>(rows)[i], 0);
  else return load1(rows, i, kBf16 ? TRIS_DTYPE_BF16 : TRIS_DTYPE_F16);
}

// What a piece's sums at dimensions d and d + 1 are where they came out as NaN and the sum of its weights is a number
// above zero: a weight's 16-bit part that is zero has made an infinite value NaN.  By the formula every finite score has a
// weight above zero, so that the sum is infinite with the sign of its infinite values; NaN if they have both, if one has
// a score of -infinity, or if a value is NaN itself.  (Such a score shows in the key alone: with an infinity or NaN in
// the query no score is finite, and a score of infinity or NaN is one of the sum too.)  131072 tokens with one row of
// infinities: the call 142 us, 50 without.  Calls without any pay 0 to 2 % (8.7 / 8.9 us for 1000 tokens in a graph,
// 52.1 / 52.5 for 128k); a second pass over the tiles with all operands in registers cost them 1 to 5 %.
template <int kDim, bool kBf16, bool kE4m3>
__device__ __forceinline__ float2 infinite_sums(const AttentionArgs& a, const Piece& p, int kvh, int d) {
  const auto& c = a.c;
  const int32_t* table = c.block_table + p.b * c.table_stride;
  bool up[2] = {false, false}, down[2] = {false, false}, nan[2] = {false, false};
#pragma unroll 1
  for (int key = max(p.first, p.t0 * kTileKeys), end = min(p.n, p.t1 * kTileKeys); key < end; ++key) {
    const int i = a.page_of(key), slot = key - i * c.page_size;
    const int64_t page = table[i];
    if (page < 0 || page >= c.num_pages) continue;
    const int64_t at = page * c.v_page_stride + kvh * c.v_head_stride + slot * c.v_slot_stride + d;
    float scale = 1.0f;
    if constexpr (kE4m3)
      scale = c.v_scale[page * c.v_scale_page_stride + kvh * c.v_scale_head_stride + slot * c.v_scale_slot_stride];
    const float v[2] = {element<kBf16, kE4m3>(c.v, at) * scale, element<kBf16, kE4m3>(c.v, at + 1) * scale};
    if (fabsf(v[0]) < INFINITY && fabsf(v[1]) < INFINITY) continue;
    bool finite = true;
    if constexpr (kE4m3) {
      finite = fabsf(c.k_scale[page * c.k_scale_page_stride + kvh * c.k_scale_head_stride +
                               slot * c.k_scale_slot_stride]) < INFINITY;
    } else {
      const int64_t row = page * c.k_page_stride + kvh * c.k_head_stride + slot * c.k_slot_stride;
#pragma unroll 1
      for (int e = 0; e < kDim; ++e) finite &= fabsf(element<kBf16, false>(c.k, row + e)) < INFINITY;
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      up[t] |= v[t] == INFINITY;
      down[t] |= v[t] == -INFINITY;
      nan[t] |= v[t] != v[t] || (fabsf(v[t]) == INFINITY && !finite);
    }
  }
  const auto sum = [&](int t) { return nan[t] || up[t] == down[t] ? __builtin_nanf("") : up[t] ? INFINITY : -INFINITY; };
  return make_float2(sum(0), sum(1));
}

// The scores of a (sequence, head group): tile by tile, in each its halves of 16 keys, in each the group's heads, so that
// a wavefront's store is one stretch of memory (64 on e4m3 199 us, 202 with a row for each head).
__device__ __forceinline__ float* score_block(const AttentionArgs& a, int b, int kvh, int head0) {
  return a.scores + ((static_cast<int64_t>(b) * a.c.kv_heads + kvh) * a.group + head0) * a.score_row;
}

// The powers of two that the weights and their sum are taken larger by (see the probabilities below).
__host__ __device__ constexpr float weight_shift(bool bf16, bool e4m3) { return e4m3 ? 0.0f : bf16 ? -16.0f : 15.0f; }

// The wavefronts' sums of a piece joined under the workgroup's maximum: to the output, or to the piece's slot.
// lds: [kWaves][tile_heads][head_dim + 4] sums, then [kWaves][16] maxima and sums.
template <int kDim, bool kBf16, bool kE4m3, bool kWeights>
__device__ __forceinline__ void write_piece(const AttentionArgs& a, const Piece& p, int thread, float m, float l,
                                            const f32x4* acc, float* lds) {
  constexpr int kRun = kDim < 128 ? kDim / 16 : 8;
  constexpr int kRuns = kDim / 16 / kRun;
  constexpr int kPad = kDim + 4;
  const int col = thread % 16, g = thread % kWave / 16, wave = uniform(thread / kWave);
  const int kvh = p.hg / a.head_tiles, head0 = (p.hg % a.head_tiles) * kHeadTile;
  const int heads = min(kHeadTile, a.group - head0);
  l = across_groups(l, [](float u, float v) { return u + v; });
  float* sh_o = lds;
  float* sh_m = lds + kWaves * a.tile_heads * kPad;
  float* sh_l = sh_m + kWaves * kHeadTile;
  if (g == 0) {
    sh_m[wave * kHeadTile + col] = m;
    sh_l[wave * kHeadTile + col] = l;
  }
  if (col < heads) {
    float* o = sh_o + (wave * a.tile_heads + col) * kPad;
#pragma unroll
    for (int c = 0; c < kRuns; ++c) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
#pragma unroll
        for (int e = 0; e < kRun; e += 4) {
          const int i = c * kRun + e;
          *reinterpret_cast<f32x4*>(o + c * 16 * kRun + (g * 4 + r) * kRun + e) =
              f32x4{acc[i][r], acc[i + 1][r], acc[i + 2][r], acc[i + 3][r]};
        }
      }
    }
  }
  __syncthreads();
  const int64_t row0 = static_cast<int64_t>(p.slot) * a.tile_heads;
  uint32_t redo = 0;
  for (int i = thread * 2; i < heads * kDim; i += kWaves * kWave * 2) {
    const int h = i / kDim, d = i % kDim;
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < kWaves; ++u) top = fmaxf(top, sh_m[u * kHeadTile + h]);
    const float base = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f, y0 = 0.0f, y1 = 0.0f;
#pragma unroll
    for (int u = 0; u < kWaves; ++u) {
      const float f = __builtin_amdgcn_exp2f(sh_m[u * kHeadTile + h] - base);
      const float* o = sh_o + (u * a.tile_heads + h) * kPad + d;
      sum += sh_l[u * kHeadTile + h] * f;
      y0 += o[0] * f;
      y1 += o[1] * f;
    }
    if (p.whole) {
      if (kWeights && d == 0)
        a.whole_ml[static_cast<int64_t>(p.b) * a.q_heads + kvh * a.group + head0 + h] = make_float2(top, sum);
      const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
      uint16_t* dst = a.out + p.b * a.out_seq + (kvh * a.group + head0 + h) * a.out_head + d;
      *reinterpret_cast<uint32_t*>(dst) = kBf16 ? pack_bf16_rne(y0 * f, y1 * f) : pack_f16_rne(y0 * f, y1 * f);
    } else {
      *reinterpret_cast<float2*>(a.part_o + (row0 + h) * kDim + d) = make_float2(y0, y1);
      if (d == 0) a.part_ml[row0 + h] = make_float2(top, sum);
    }
    if ((y0 != y0 || y1 != y1) && sum > 0.0f && sum < INFINITY) redo |= 1u << i / (kWaves * kWave * 2);
  }
  if (!__any(redo != 0)) return;
#pragma unroll 1
  for (int i = thread * 2; i < heads * kDim; i += kWaves * kWave * 2, redo >>= 1) {
    if (!(redo & 1)) continue;
    const int h = i / kDim, d = i % kDim;
    const float2 y = infinite_sums<kDim, kBf16, kE4m3>(a, p, kvh, d);
    if (p.whole) {
      uint16_t* dst = a.out + p.b * a.out_seq + (kvh * a.group + head0 + h) * a.out_head + d;
      const int32_t type = kBf16 ? TRIS_DTYPE_BF16 : TRIS_DTYPE_F16;
      if (isnan(load1(dst, 0, type))) store1(dst, 0, y.x, type);
      if (isnan(load1(dst, 1, type))) store1(dst, 1, y.y, type);
    } else {
      float* dst = a.part_o + (row0 + h) * kDim + d;
      if (isnan(dst[0])) dst[0] = y.x;
      if (isnan(dst[1])) dst[1] = y.y;
    }
  }
}

// kRowRuns: every 16 keys of a tile lie in one page (page_size a multiple of 16; with e4m3, scale rows that can be read
// four at a time), so that page numbers and row addresses are the same for the whole wavefront; else each lane looks
// up one key and hands its rows' addresses around (of the same calls, with runs / by lanes: 128k 50.9 / 55.5 us, windowed
// 83.8 / 86.4, 64 on e4m3 138 / 139, ragged 24.2 / 25.4).
template <int kDim, bool kBf16, bool kE4m3, bool kRowRuns, bool kWeights>
__device__ __forceinline__ void attend_piece(const AttentionArgs& a, const Piece& p, int thread, u32x4 (*sh_q)[kWave],
                                             float* lds) {
  constexpr bool kBf16V = kBf16 || kE4m3;           // type of the value product (see the probabilities below)
  constexpr int kRun = kDim < 128 ? kDim / 16 : 8;  // dimensions of one of a lane's runs of a value row
  constexpr int kRuns = kDim / 16 / kRun;
  constexpr int kSize = kE4m3 ? 1 : 2;
  constexpr int kKLoads = kDim * kSize / 64;        // 16-byte loads of a lane for one key row's quarter
  constexpr int kVWords = kRun * kSize / 4;         // words of a run
  constexpr bool kQueryInLds = query_in_lds(kDim);
  const int n = p.n, first = p.first, t1 = p.t1, t_end = n > 0 ? t1 : 0;
  const int kvh = p.hg / a.head_tiles, head0 = (p.hg % a.head_tiles) * kHeadTile;
  const int heads = min(kHeadTile, a.group - head0);
  const int wave = uniform(thread / kWave), lane = thread % kWave, col = lane % 16, g = lane / 16;

  // in bytes
  const int64_t k_page = a.c.k_page_stride * kSize, v_page = a.c.v_page_stride * kSize;
  const int64_t ks_page = a.c.k_scale_page_stride * 4, vs_page = a.c.v_scale_page_stride * 4;
  const int k_slot = static_cast<int>(a.c.k_slot_stride) * kSize, v_slot = static_cast<int>(a.c.v_slot_stride) * kSize;
  const int ks_slot = static_cast<int>(a.c.k_scale_slot_stride) * 4, vs_slot = static_cast<int>(a.c.v_scale_slot_stride) * 4;

  // The query operand: head col, the dimensions that the K operand's lane has.  At 256 dimensions it would push the
  // tiles' loads out of the registers (it is 32 of them), so there it stays in LDS, read when it is used (wide: 30.0
  // us, 36.2 with it in registers; at 128 dimensions both ways take the same time).
  u32x4 q[kQueryInLds ? 1 : kDim / 32];
  const auto query = [&](int i) {
    const int d = kE4m3 ? (i / 2) * 64 + g * 16 + (i % 2) * 8 : i * 32 + g * 8;
    return col < heads ? *reinterpret_cast<const u32x4*>(a.q + p.b * a.q_seq + (kvh * a.group + head0 + col) * a.q_head + d)
                       : u32x4{0, 0, 0, 0};
  };
  if constexpr (kQueryInLds) {
    for (int i = wave; i < kDim / 32; i += kWaves) sh_q[i][lane] = query(i);
    __syncthreads();
  } else {
#pragma unroll
    for (int i = 0; i < kDim / 32; ++i) q[i] = query(i);
  }

  const char* kbase = static_cast<const char*>(a.c.k) + kvh * a.c.k_head_stride * kSize;
  const char* vbase = static_cast<const char*>(a.c.v) + kvh * a.c.v_head_stride * kSize;
  const char* ksbase = reinterpret_cast<const char*>(a.c.k_scale) + kvh * a.c.k_scale_head_stride * 4;
  const char* vsbase = reinterpret_cast<const char*>(a.c.v_scale) + kvh * a.c.v_scale_head_stride * 4;
  const int32_t* table = a.c.block_table + p.b * a.c.table_stride;
  // wavefronts take the workgroup's tiles in turn, also over the pieces
  int tile = p.t0 + ((wave - p.at) & (kWaves - 1));

  // Page numbers run ahead of the rows, so that no row waits for its page: with kRowRuns lane 2 i + t holds the block
  // table's entry of half t of the wavefront's i-th tile from `ids0`, 32 tiles a load and the next 32 behind them; else lane
  // 32 i + k that of key k of the next tile.  Entries past the table's end read its last one; all are checked where
  // they are used.
  const auto entry = [&](int key) { return table[min(a.page_of(key), a.c.max_pages - 1)]; };
  const auto fetch_ids = [&](int from) {
    if constexpr (kRowRuns) return entry((from + lane / 2 * kWaves) * kTileKeys + lane % 2 * 16);
    else return entry(from * kTileKeys + lane % kTileKeys);
  };
  // the pages of one tile: of its halves, or of the key that the lane looked up, -1 where there is none; and of that
  // key, where its rows are and its scales (page 0's where it has none: it is masked)
  struct Pages {
    int id[2];
    int64_t k, v;
    float ks, vs;
  };
  const auto checked = [&](int key, int id, int of_tile) {
    return of_tile < t1 && key < n && static_cast<uint32_t>(id) < static_cast<uint32_t>(a.c.num_pages) ? id : -1;
  };
  const auto pages_of = [&](int of_tile, int ids, int i) {
    Pages pg;
    if constexpr (kRowRuns) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
        pg.id[t] = checked(of_tile * kTileKeys + t * 16, __builtin_amdgcn_readlane(ids, 2 * i + t), of_tile);
    } else {
      const int key = of_tile * kTileKeys + lane % kTileKeys;
      pg.id[0] = checked(key, ids, of_tile);
      const int64_t page = max(pg.id[0], 0), slot = key - a.page_of(key) * a.c.page_size;
      pg.k = page * k_page + slot * k_slot;
      pg.v = page * v_page + slot * v_slot;
      if constexpr (kE4m3) {
        pg.ks = load_global<float, false>(ksbase + page * ks_page, static_cast<uint32_t>(slot * ks_slot));
        pg.vs = load_global<float, false>(vsbase + page * vs_page, static_cast<uint32_t>(slot * vs_slot));
      }
    }
    return pg;
  };
  // With kRowRuns: one half's 16 rows as a buffer that ends with the sequence, empty without a page or past the workgroup's
  // tiles: rows outside read as zeros, without a memory access and without a branch.
  const auto half_rows = [&](const char* base, int64_t page_stride, int slot_bytes, int of_tile, const Pages& pg, int t) {
    const int key = of_tile * kTileKeys + t * 16, page = pg.id[t];
    const int slot = key - a.page_of(key) * a.c.page_size, rows = page >= 0 ? min(16, n - key) : 0;
    return make_rsrc(base + max(page, 0) * page_stride + static_cast<int64_t>(slot) * slot_bytes,
                     static_cast<uint32_t>(rows * slot_bytes));
  };
  // Else: a row of the tile's k-th key, by the lane that looked it up.
  const auto of_key = [&](int64_t offset, int k) {
    const int lo = __shfl(static_cast<int>(offset), k), hi = __shfl(static_cast<int>(offset >> 32), k);
    return static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(hi)) << 32 | static_cast<uint32_t>(lo));
  };

  u32x4 kr[2][kKLoads] = {};
  uint32_t vr[8][kRuns * kVWords] = {};
  float ks[8] = {}, vs[8] = {};
  const auto load_k = [&](int tile, const Pages& pg) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      if constexpr (kRowRuns) {
        const __amdgpu_buffer_rsrc_t rows = half_rows(kbase, k_page, k_slot, tile, pg, t);
#pragma unroll
        for (int i = 0; i < kKLoads; ++i)
          kr[t][i] = __builtin_amdgcn_raw_buffer_load_b128(rows, col * k_slot + g * 16, i * 64, kLoadOnce);
        if constexpr (kE4m3) {
          const __amdgpu_buffer_rsrc_t scales = half_rows(ksbase, ks_page, 4, tile, pg, t);
          const u32x4 s = __builtin_amdgcn_raw_buffer_load_b128(scales, g * 16, 0, 0);
#pragma unroll
          for (int r = 0; r < 4; ++r) ks[t * 4 + r] = __uint_as_float(s[r]);
        }
      } else {
        const char* row = kbase + of_key(pg.k, t * 16 + col);
#pragma unroll
        for (int i = 0; i < kKLoads; ++i)
          kr[t][i] = load_global<u32x4, false>(row, static_cast<uint32_t>(g * 16 + i * 64));
      }
    }
  };
  const auto load_v = [&](int tile, const Pages& pg) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      __amdgpu_buffer_rsrc_t rows, scales;
      if constexpr (kRowRuns) rows = half_rows(vbase, v_page, v_slot, tile, pg, t);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int j = t * 4 + r;
        const char* row = vbase;
        if constexpr (!kRowRuns) row += of_key(pg.v, t * 16 + g * 4 + r);
#pragma unroll
        for (int c = 0; c < kRuns; ++c) {
          uint32_t* dst = vr[j] + c * kVWords;
          const int in_row = col * kRun * kSize + c * 16 * kRun * kSize;
          if constexpr (kRowRuns) {
            const int at_row = (g * 4 + r) * v_slot + in_row;
            if constexpr (kVWords == 4)
              *reinterpret_cast<u32x4*>(dst) = __builtin_amdgcn_raw_buffer_load_b128(rows, at_row, 0, kLoadOnce);
            else if constexpr (kVWords == 2)
              *reinterpret_cast<u32x2*>(dst) = __builtin_amdgcn_raw_buffer_load_b64(rows, at_row, 0, kLoadOnce);
            else
              *dst = __builtin_amdgcn_raw_buffer_load_b32(rows, at_row, 0, kLoadOnce);
          } else {
            const uint32_t at_row = static_cast<uint32_t>(in_row);
            if constexpr (kVWords == 4) *reinterpret_cast<u32x4*>(dst) = load_global<u32x4, true>(row, at_row);
            else if constexpr (kVWords == 2) *reinterpret_cast<u32x2*>(dst) = load_global<u32x2, true>(row, at_row);
            else *dst = load_global<uint32_t, true>(row, at_row);
          }
        }
      }
      if constexpr (kE4m3 && kRowRuns) {
        scales = half_rows(vsbase, vs_page, 4, tile, pg, t);
        const u32x4 s = __builtin_amdgcn_raw_buffer_load_b128(scales, g * 16, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r) vs[t * 4 + r] = __uint_as_float(s[r]);
      }
    }
  };

  float* const scores = kWeights ? score_block(a, p.b, kvh, head0) : nullptr;
  const int score_at = col < heads ? (col * 16 + g * 4) * 4 : INT32_MAX;  // the lane's four keys of its head, in bytes

  float m = -INFINITY, l = 0.0f;
  f32x4 acc[kRuns * kRun];
#pragma unroll
  for (int i = 0; i < kRuns * kRun; ++i) acc[i] = f32x4{0, 0, 0, 0};

  // A tile's keys and values are loaded while the tile before it is computed: the next tile's keys are asked for when
  // this one's have been used, the values likewise, without a branch (past the last tile from empty buffers, by lanes
  // rows of page 0): behind one, the compiler waits for every load in flight before it uses the values.
  const int tile0 = tile;
  Pages cur = {}, nxt = {};
  int ids = 0, ahead = 0;
  if (tile < t_end) {
    ids = fetch_ids(tile);
    ahead = fetch_ids(tile + (kRowRuns ? kWave / 2 : 1) * kWaves);
    cur = pages_of(tile, ids, 0);
    load_k(tile, cur);
    load_v(tile, cur);
  }
  for (int i = 1; tile < t_end; ++i, tile += kWaves) {
    if constexpr (kRowRuns) {
      if (i % (kWave / 2) == 0) {
        ids = ahead;
        ahead = fetch_ids(tile0 + (i + kWave / 2) * kWaves);
      }
      nxt = pages_of(tile + kWaves, ids, i % (kWave / 2));
    } else {
      nxt = pages_of(tile + kWaves, ahead, 0);
      ahead = fetch_ids(tile + 2 * kWaves);
    }
    int q_lane = lane;
    if constexpr (kQueryInLds) asm volatile("" : "+v"(q_lane));  // read anew for each tile, not kept
    f32x4 s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      s[t] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < kDim / 32; ++i) {
        u32x4 k;
        if constexpr (kE4m3) {
          const u32x4 w = kr[t][i / 2];
          const uint32_t w0 = w[(i % 2) * 2], w1 = w[(i % 2) * 2 + 1];
          k = u32x4{from_e4m3<kBf16, false>(w0), from_e4m3<kBf16, true>(w0), from_e4m3<kBf16, false>(w1),
                    from_e4m3<kBf16, true>(w1)};
        } else {
          k = kr[t][i];
        }
        s[t] = mfma<kBf16>(k, kQueryInLds ? sh_q[i][q_lane] : q[kQueryInLds ? 0 : i], s[t]);
      }
    }
    if constexpr (kE4m3 && !kRowRuns) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int k = j / 4 * 16 + g * 4 + j % 4;
        ks[j] = __shfl(cur.ks, k);
        vs[j] = __shfl(cur.vs, k);
      }
    }
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = s[j / 4][j % 4] * a.scale_log2;
      if constexpr (kE4m3) x[j] *= ks[j];
    }
    // keys outside the sequence, before its window or without a page
    const int key0 = tile * kTileKeys;
    bool edge = key0 < first || key0 + kTileKeys > n;
    if constexpr (kRowRuns) edge = edge || cur.id[0] < 0 || cur.id[1] < 0;
    else edge = edge || __any(cur.id[0] < 0);
    bool valid[8];
    if (edge) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int k = j / 4 * 16 + g * 4 + j % 4;
        const int id = kRowRuns ? cur.id[j / 4] : __shfl(cur.id[0], k);  // (from any lane: before the lane's own test)
        valid[j] = key0 + k >= first && key0 + k < n && id >= 0;
        x[j] = valid[j] ? x[j] : -INFINITY;
      }
    }
    // (a lane without a head: outside the buffer, without a branch, which would make the loads in flight wait: wide 37.9 us,
    // 39.1 with one)
    if constexpr (kWeights) {
      const __amdgpu_buffer_rsrc_t rows = make_rsrc(scores + static_cast<int64_t>(key0) * heads, heads * 128);
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, f32x4{x[0], x[1], x[2], x[3]}), rows, score_at, 0, 0);
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, f32x4{x[4], x[5], x[6], x[7]}), rows, score_at,
                                             heads * 64, 0);
    }
    load_k(tile + kWaves, nxt);

    float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
    if (__any(top > m)) {
      const float now = across_groups(fmaxf(m, top), [](float u, float w) { return fmaxf(u, w); });
      const float f = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - now);
      m = now;
      l *= f;
#pragma unroll
      for (int i = 0; i < kRuns * kRun; ++i) acc[i] *= f;
    }
    // The probabilities enter the value product as three 16-bit parts, each what the one before left, which together are
    // their 24 bits (in fp16 down to 2^-39 of the head's largest): the result has one rounding to speak of, the output's.
    // (Three parts / two: 128k 52.0 / 52.1 us, windowed 83.5 / 83.3, 64 on e4m3 142.4 / 141.6: the matrix cores wait for
    // memory.)  They are taken 2^kShift times as large, the sum too, so that it cancels: in fp16 a long tail far below
    // the maximum would lose its bits to the subnormals otherwise, and of bf16 values near the type's largest two would
    // pass fp32's range.  An 8-bit cache's product runs in bf16, whose range takes any scale; its elements are exact in
    // either type, and a small scale leaves no room for a shift.
    constexpr float kShift = weight_shift(kBf16, kE4m3);
    const float base = (m == -INFINITY ? 0.0f : m) - kShift;
    float pr[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      pr[j] = __builtin_amdgcn_exp2f(x[j] - base);
      l += pr[j];
      if constexpr (kE4m3) pr[j] *= vs[j];
    }
    if (edge) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        pr[j] = valid[j] ? pr[j] : 0.0f;
        // (a buffer's end has done this for rows past the sequence)
        if (!kRowRuns || key0 < first) {
#pragma unroll
          for (int i = 0; i < kRuns * kVWords; ++i) vr[j][i] = valid[j] ? vr[j][i] : 0u;
        }
      }
    }
    u32x4 part[3];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float w0 = pr[2 * i], w1 = pr[2 * i + 1];
#pragma unroll
      for (int u = 0; u < 3; ++u) {
        if constexpr (kBf16V) {
          const uint32_t u0 = __float_as_uint(w0), u1 = __float_as_uint(w1);
          part[u][i] = __builtin_amdgcn_perm(u1, u0, 0x07060302u);
          w0 -= __uint_as_float(u0 & 0xFFFF0000u);
          w1 -= __uint_as_float(u1 & 0xFFFF0000u);
        } else {
          const auto h = __builtin_amdgcn_cvt_pkrtz(w0, w1);
          part[u][i] = __builtin_bit_cast(uint32_t, h);
          w0 -= static_cast<float>(h[0]);
          w1 -= static_cast<float>(h[1]);
        }
      }
    }
#pragma unroll
    for (int c = 0; c < kRuns; ++c) {
#pragma unroll
      for (int e = 0; e < kRun; e += 2) {
        uint32_t word[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if constexpr (kE4m3) {
            const uint32_t v = vr[j][c * kVWords + e / 4];
            word[j] = e % 4 == 0 ? from_e4m3<true, false>(v) : from_e4m3<true, true>(v);
          } else {
            word[j] = vr[j][c * kVWords + e / 2];
          }
        }
#pragma unroll
        for (int odd = 0; odd < 2; ++odd) {
          const uint32_t sel = odd ? 0x07060302u : 0x05040100u;
          const u32x4 v = {__builtin_amdgcn_perm(word[1], word[0], sel), __builtin_amdgcn_perm(word[3], word[2], sel),
                           __builtin_amdgcn_perm(word[5], word[4], sel), __builtin_amdgcn_perm(word[7], word[6], sel)};
          f32x4& o = acc[c * kRun + e + odd];
#pragma unroll
          for (int u = 0; u < 3; ++u) o = mfma<kBf16V>(v, part[u], o);
        }
      }
    }
    load_v(tile + kWaves, nxt);
    cur = nxt;
  }

  asm volatile("" : "+v"(thread));  // (what follows takes the lane's number anew too)
  write_piece<kDim, kBf16, kE4m3, kWeights>(a, p, thread, m, l, acc, lds);
}

// The maximum and sum of two sets of keys together.
__device__ __forceinline__ float2 joined(float2 x, float2 y) {
  const float top = fmaxf(x.x, y.x), base = top == -INFINITY ? 0.0f : top;
  return make_float2(top, x.y * __builtin_amdgcn_exp2f(x.x - base) + y.y * __builtin_amdgcn_exp2f(y.x - base));
}

// Adds the weights of a piece's keys (tiles [t0, t1) of sequence b's n positions from `first` on) to the sums of their kv
// head, from the scores that the attention left, for all query heads of the kv head.  stats: LDS for 1 + kWaves float2 of each.
// A thread has four keys; the scores of eight heads are asked for a step ahead of their use, the first ones before the
// statistics are known.  (The sums and pages asked for with them: no difference.)
__device__ __forceinline__ void sum_weights(const AttentionArgs& a, int b, int kvh, int n, int first, int t0, int t1,
                                            float shift, float2* stats) {
  const bool sums4 = a.sums4 != 0;
  constexpr int kStep = 8;
  const int thread = threadIdx.x, wave = uniform(thread / kWave), lane = thread % kWave;
  const int32_t* table = a.c.block_table + b * a.c.table_stride;
  float* const sums = a.weight_sum + b * a.sum_seq + kvh * a.sum_head;
  const float* const scores = score_block(a, b, kvh, 0);
  const int end = min(n, t1 * kTileKeys);
  int key = t0 * kTileKeys + thread * 4, h0 = 0;
  f32x4 x[kStep], ahead[kStep];
  // the scores of four keys and heads from h on, of the kv head's last ones again past them
  const auto load = [&](int k, int h, f32x4* to) {
    const int head0 = h / kHeadTile * kHeadTile, heads = min(kHeadTile, a.group - head0);
    const float* from = scores + head0 * a.score_row + static_cast<int64_t>(k / kTileKeys * kTileKeys) * heads +
                        k / 16 % 2 * heads * 16 + k % 16;
#pragma unroll
    for (int i = 0; i < kStep; ++i)
      to[i] = *reinterpret_cast<const f32x4*>(from + min(h - head0 + i, heads - 1) * 16);
  };
  if (key < end) load(key, 0, x);

  // Each head's maximum and sum over the pieces.  Of few pieces a wavefront takes a head, a lane a piece; of many a lane takes
  // one head and every sixteenth piece (131072 tokens, 192 pieces: the launch 12.0 us, 13.3 the other way; 16 ragged, 6
  // pieces, 8.5, 8.9 the other way).
  const auto owners = [&](int tile) {
    return a.owners == nullptr ? make_int2(0, 0) : a.owners[(b * a.c.kv_heads + kvh) * a.head_tiles + tile];
  };
  const auto part = [&](int w, int2 own, int col) {
    return a.part_ml[static_cast<int64_t>(2 * w + (w == own.x)) * a.tile_heads + col];
  };
  const float2* const whole = a.whole_ml + static_cast<int64_t>(b) * a.q_heads + kvh * a.group;
  const auto to_stats = [&](int h, float top, float l) {
    stats[h] = make_float2((top == -INFINITY ? 0.0f : top) - shift, l == 0.0f ? 0.0f : 1.0f / l);
  };
  const int2 own0 = owners(0);
  if (own0.y - own0.x < kWave) {
    for (int h = wave; h < a.group; h += kWaves) {
      const int2 own = h < kHeadTile ? own0 : owners(h / kHeadTile);
      if (own.x == own.y) {
        const float2 ml = whole[h];
        if (lane == 0) to_stats(h, ml.x, ml.y);
      } else {
        float2 ml = {-INFINITY, 0.0f};
        for (int w = own.x + lane; w <= own.y; w += kWave) ml = joined(ml, part(w, own, h % kHeadTile));
        const float top = wave_max_f32(ml.x);
        const float l = wave_sum_f32(ml.y * __builtin_amdgcn_exp2f(ml.x - (top == -INFINITY ? 0.0f : top)));
        if (lane == 0) to_stats(h, top, l);
      }
    }
  } else {
    float2* const shares = stats + a.group;  // [kWaves][group]
    for (int tile = 0; tile < a.head_tiles; ++tile) {
      const int col = lane % kHeadTile, heads = min(kHeadTile, a.group - tile * kHeadTile);
      const int2 own = owners(tile);
      float2 ml = {-INFINITY, 0.0f};
      if (col < heads && own.x == own.y) {
        if (thread < kHeadTile) ml = whole[tile * kHeadTile + col];
      } else if (col < heads) {
#pragma unroll 4
        for (int w = own.x + thread / kHeadTile; w <= own.y; w += kWaves * kWave / kHeadTile)
          ml = joined(ml, part(w, own, col));
      }
      const float top = across_groups(ml.x, [](float u, float v) { return fmaxf(u, v); });
      const float l = across_groups(ml.y * __builtin_amdgcn_exp2f(ml.x - (top == -INFINITY ? 0.0f : top)),
                                    [](float u, float v) { return u + v; });
      if (lane < heads) shares[wave * a.group + tile * kHeadTile + lane] = make_float2(top, l);
    }
    __syncthreads();
    for (int h = thread; h < a.group; h += kWaves * kWave) {
      float2 ml = shares[h];
#pragma unroll
      for (int u = 1; u < kWaves; ++u) ml = joined(ml, shares[u * a.group + h]);
      to_stats(h, ml.x, ml.y);
    }
  }
  __syncthreads();

  f32x4 weight = {0, 0, 0, 0};
  while (key < end) {
    const bool last = h0 + kStep >= a.group;
    const int key2 = last ? key + kWaves * kWave * 4 : key, h2 = last ? 0 : h0 + kStep;
    if (key2 < end) load(key2, h2, ahead);
#pragma unroll
    for (int i = 0; i < kStep; ++i) {
      if (h0 + i < a.group) {
        const float2 of = stats[h0 + i];
#pragma unroll
        for (int e = 0; e < 4; ++e) weight[e] += __builtin_amdgcn_exp2f(x[i][e] - of.x) * of.y;
      }
    }
    if (last) {
      const auto valid = [&](int k) {
        return k >= first && k < n && static_cast<uint32_t>(table[a.page_of(k)]) < static_cast<uint32_t>(a.c.num_pages);
      };
      const bool use[4] = {valid(key), valid(key + 1), valid(key + 2), valid(key + 3)};
      if (sums4 && use[0] && use[1] && use[2] && use[3]) {
        f32x4* to = reinterpret_cast<f32x4*>(sums + key);
        *to = *to + weight;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (use[e]) sums[key + e] += weight[e];
      }
      weight = f32x4{0, 0, 0, 0};
    }
    key = key2;
    h0 = h2;
#pragma unroll
    for (int i = 0; i < kStep; ++i) x[i] = ahead[i];
  }
}

template <int kDim, bool kBf16, bool kE4m3, bool kRowRuns, bool kWeights>
__global__ __launch_bounds__(kWaves * kWave, resident(kDim)) void attention_decode_kernel(const AttentionArgs args) {
  __shared__ u32x4 sh_q[query_in_lds(kDim) ? kDim / 32 : 1][kWave];
  extern __shared__ float lds[];
  const int head_groups = args.c.kv_heads * args.head_tiles, w = blockIdx.x;
  Stretch st;
  if (!(args.owners == nullptr ? own_stretch(args, head_groups, w, &st) : line_stretch(args, head_groups, w, &st)))
    return;
  int at = st.at, begin = st.begin, b = st.b, n = st.n;
  const int stop = st.stop;
  // one piece of a (sequence, head group) after the other
  while (at < stop && b < args.c.batch) {
    // What a piece needs of the arguments and of the lane's number is taken anew for each: kept in registers from piece
    // to piece, it would cost the tiles' loop a third of its wavefronts.
    int thread = threadIdx.x;
    KernelArgs fresh = (KernelArgs)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+v"(thread), "+s"(fresh));
    const AttentionArgs& a = *(const AttentionArgs*)fresh;
    const int first = range_begin(a, n), tiles = range_tiles(n, first), span = tiles + kPieceCost;
    const int hg = (at - begin) / span, from = at - begin - hg * span;
    if (hg == head_groups) {  // the next sequence
      begin = at;
      n = uniform(sequence_length(a, ++b));
      continue;
    }
    if (from >= tiles) {  // between two head groups
      at += span - from;
      continue;
    }
    if (a.owners != nullptr && from == 0 && thread == 0)
      a.owners[b * head_groups + hg] = make_int2(w, st.line.owner(at + tiles - 1));
    const int count = min(tiles - from, stop - at), t0 = first / kTileKeys + from;
    // a piece that begins its (sequence, head group) and is not all of it ends its workgroup's stretch: the second slot
    const Piece p{b, n, first, hg, t0, t0 + count, at, 2 * w + (from == 0), count == tiles};
    attend_piece<kDim, kBf16, kE4m3, kRowRuns, kWeights>(a, p, thread, sh_q, lds);
    at += count;
    __syncthreads();  // the next piece's sums go where this one's are read
    if constexpr (kWeights) {
      if (own_weights(a) && n > 0)
        sum_weights(a, b, hg, n, first, t0, t0 + count, weight_shift(kBf16, kE4m3), reinterpret_cast<float2*>(lds));
    }
  }
}

// Pieces of a (sequence, head group) on average, from which a join takes 16 or 4 wavefronts for the same dimensions (16 /
// 4 / 1 together: 192 pieces, 128k, 50.8 / 51.0 / 54.4 us; 32 pieces, wide, 33.0 / 30.0 / 30.7; 9 pieces, 1000 tokens,
// 9.7 / 9.4 / 9.1; 6 pieces, ragged, 30.6 / 24.5 / 24.2; 1.5 pieces, 64 on e4m3, 177 / 145 / 138).
constexpr int kJoinMany = 64, kJoinSome = 16;

// A lane's share of a join: the running maximum, sum and four dimensions' sums, and another's added to them.
struct Part {
  float m, l;
  f32x4 o;
  __device__ __forceinline__ void add(float m2, float l2, f32x4 o2) {
    const float top = fmaxf(m, m2), base = top == -INFINITY ? 0.0f : top;
    const float f = __builtin_amdgcn_exp2f(m - base), f2 = __builtin_amdgcn_exp2f(m2 - base);
    m = top;
    l = l * f + l2 * f2;
    o = o * f + o2 * f2;
  }
  // over the wavefront's lanes of the same dimensions
  __device__ __forceinline__ void across() {
#pragma unroll
    for (int d = 8; d < kWave; d *= 2) {
      const f32x4 o2 = {__shfl_xor(o[0], d), __shfl_xor(o[1], d), __shfl_xor(o[2], d), __shfl_xor(o[3], d)};
      const float m2 = __shfl_xor(m, d), l2 = __shfl_xor(l, d);
      // (in the same order on both sides, so that both get the same bits)
      if (threadIdx.x & d) {
        Part other{m2, l2, o2};
        other.add(m, l, o);
        *this = other;
      } else {
        add(m2, l2, o2);
      }
    }
  }
};

// Joins the pieces of one (sequence, query head), 32 dimensions a wavefront: eight lanes a piece, eight pieces at a time.
// kTogether: 16 or 4 shares of the pieces for the same dimensions, by kJoinWaves wavefronts, or (1) four wavefronts on
// dimensions of their own.
template <int kDim, bool kBf16, int kTogether, int kJoinWaves>
__device__ __forceinline__ void join_pieces(const AttentionArgs& a, int block) {
  constexpr int kParts = kDim / 32;
  constexpr bool kMany = kTogether > 1;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const int unit = block * (kMany ? 1 : 4) + (kMany ? 0 : wave);
  const int row = unit / kParts, d = unit % kParts * 32 + lane % 8 * 4;
  const int b = row / a.q_heads, h = row % a.q_heads;
  if (b >= a.c.batch) return;
  const int hg = h / a.group * a.head_tiles + h % a.group / kHeadTile, in = h % a.group % kHeadTile;
  const int2 owners = a.owners[b * (a.c.kv_heads * a.head_tiles) + hg];
  if (owners.x == owners.y) return;
  constexpr int kShares = kMany ? kTogether / kJoinWaves : 1;  // of a wavefront
  Part p[kShares];
#pragma unroll
  for (int u = 0; u < kShares; ++u) {
    p[u] = Part{-INFINITY, 0.0f, f32x4{0, 0, 0, 0}};
#pragma unroll 2
    for (int w = owners.x + (kMany ? (wave + u * kJoinWaves) * 8 : 0) + lane / 8; w <= owners.y; w += 8 * kTogether) {
      const int64_t r = static_cast<int64_t>(2 * w + (w == owners.x)) * a.tile_heads + in;
      const float2 ml = a.part_ml[r];
      p[u].add(ml.x, ml.y, *reinterpret_cast<const f32x4*>(a.part_o + r * kDim + d));
    }
    p[u].across();
  }
  if constexpr (kMany) {
    __shared__ Part sh[kTogether][8];
#pragma unroll
    for (int u = 0; u < kShares; ++u)
      if (lane < 8) sh[wave + u * kJoinWaves][lane] = p[u];
    __syncthreads();
    if (wave != 0) return;
    p[0] = lane / 8 < kTogether ? sh[lane / 8 % kTogether][lane % 8] : Part{-INFINITY, 0.0f, f32x4{0, 0, 0, 0}};
    if constexpr (kTogether > 8) {
      const Part q = sh[lane / 8 + 8][lane % 8];
      p[0].add(q.m, q.l, q.o);
    }
    p[0].across();
  }
  if (lane >= 8) return;
  Part& sum = p[0];
  // A factor of zero has made a piece's infinite sum NaN: the weights that it stands for are above zero, so that the whole
  // is that of the infinite sums alone.
  const bool lost = sum.o[0] != sum.o[0] || sum.o[1] != sum.o[1] || sum.o[2] != sum.o[2] || sum.o[3] != sum.o[3];
  if (lost && sum.l > 0.0f && sum.l < INFINITY) {
    f32x4 infinite = {0, 0, 0, 0};
#pragma unroll 1
    for (int w = owners.x; w <= owners.y; ++w) {
      const int64_t r = static_cast<int64_t>(2 * w + (w == owners.x)) * a.tile_heads + in;
      const f32x4 o = *reinterpret_cast<const f32x4*>(a.part_o + r * kDim + d);
#pragma unroll
      for (int i = 0; i < 4; ++i) infinite[i] += fabsf(o[i]) < INFINITY ? 0.0f : o[i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) sum.o[i] = sum.o[i] != sum.o[i] && infinite[i] != 0.0f ? infinite[i] : sum.o[i];
  }
  const f32x4 y = sum.o * (sum.l == 0.0f ? 0.0f : 1.0f / sum.l);
  const uint2 packed = kBf16 ? make_uint2(pack_bf16_rne(y[0], y[1]), pack_bf16_rne(y[2], y[3]))
                             : make_uint2(pack_f16_rne(y[0], y[1]), pack_f16_rne(y[2], y[3]));
  *reinterpret_cast<uint2*>(a.out + b * a.out_seq + h * a.out_head + d) = packed;
}

template <int kDim, bool kBf16, int kTogether>
__global__ __launch_bounds__(kTogether == 16 ? 1024 : 256) void attention_join_kernel(const AttentionArgs a) {
  join_pieces<kDim, kBf16, kTogether, (kTogether == 16 ? 16 : 4)>(a, static_cast<int>(blockIdx.x));
}

// The second launch of the calls that sum the weights: a.workgroups workgroups add the weights, each those of the stretch
// that the workgroup of its number took in the first launch (of its pieces the first head group of each kv head, for all of
// them), and behind them the join's, where there is a line.  shift: weight_shift of the types.
template <int kDim, bool kBf16, int kTogether>
__global__ __launch_bounds__(kWaves * kWave) void attention_weights_kernel(const AttentionArgs a, const float shift) {
  extern __shared__ float2 stats[];
  if (blockIdx.x >= static_cast<uint32_t>(a.workgroups)) {
    join_pieces<kDim, kBf16, kTogether, kWaves>(a, static_cast<int>(blockIdx.x) - a.workgroups);
    return;
  }
  const int head_groups = a.c.kv_heads * a.head_tiles;
  Stretch st;
  if (!(a.owners == nullptr ? own_stretch(a, head_groups, blockIdx.x, &st)
                            : line_stretch(a, head_groups, blockIdx.x, &st)))
    return;
  int at = st.at, begin = st.begin, b = st.b, n = st.n;
  while (at < st.stop && b < a.c.batch) {
    const int first = range_begin(a, n), tiles = range_tiles(n, first), span = tiles + kPieceCost;
    const int hg = (at - begin) / span, from = at - begin - hg * span;
    if (hg == head_groups) {
      begin = at;
      n = uniform(sequence_length(a, ++b));
      continue;
    }
    const int count = min(tiles - from, st.stop - at);
    at += from >= tiles ? span - from : count;
    if (from >= tiles || n == 0 || hg % a.head_tiles != 0) continue;
    const int t0 = first / kTileKeys + from;
    sum_weights(a, b, hg / a.head_tiles, n, first, t0, t0 + count, shift, stats);
    __syncthreads();  // the statistics have been read
  }
}

// Positions times head_dim of a block table up to which a (sequence, head group) is one workgroup's: one launch, no
// workspace, no line; twice as many where there is one for each CU.  Only the table's width is known here, not the lengths:
// beyond, one long sequence would hold up the call.  In a graph, on the line / whole, us: one sequence of 128, 512, 1024
// with 8 kv heads of 128: 7.5 / 5.1, 8.6 / 8.4, 8.8 / 14.6 (called eagerly 14.1 / 10.1, 14.1 / 10.3, 14.4 / 14.5); 64 of
// 512, 1024 and 2048: 33 / 24, 53 / 44, 95 / 83; one of 128, 256 and 512 with 2 kv heads of 256: 11.3 / 9.4, 12.3 / 11.3,
// 12.2 / 16.1.
constexpr int64_t kNarrow = 512 * 128;

// The launch's sizes, from shapes alone.
struct AttentionShape {
  int group, head_tiles, tile_heads, workgroups;
  int64_t places;  // of the line, at most
  bool line;
};

static AttentionShape attention_shape(int64_t batch, int q_heads, int kv_heads, int head_dim, int64_t positions) {
  AttentionShape s;
  s.group = q_heads / kv_heads;
  s.head_tiles = (s.group + kHeadTile - 1) / kHeadTile;
  s.tile_heads = std::min(s.group, kHeadTile);
  const int64_t head_groups = static_cast<int64_t>(kv_heads) * s.head_tiles;
  const int64_t most = positions / kTileKeys + 2;  // of one sequence: a window may begin and end inside a tile
  s.places = batch * (most + kPieceCost) * head_groups;
  s.line = positions * head_dim > kNarrow * (batch * head_groups >= kCus ? 2 : 1);
  s.workgroups = static_cast<int>(s.line ? std::min<int64_t>(kCus * resident(head_dim), (s.places + kWaves - 1) / kWaves)
                                         : std::min<int64_t>(batch * head_groups, 2147483647LL));
  return s;
}

struct AttentionSpace {
  int64_t ml, o, bytes;
};

static AttentionSpace attention_space(const AttentionShape& s, int64_t batch, int kv_heads, int head_dim) {
  const auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
  AttentionSpace w;
  const int64_t rows = 2LL * s.workgroups * s.tile_heads;
  w.ml = up(batch * kv_heads * s.head_tiles * static_cast<int64_t>(sizeof(int2)));
  w.o = w.ml + up(rows * static_cast<int64_t>(sizeof(float2)));
  w.bytes = s.line ? w.o + rows * head_dim * static_cast<int64_t>(sizeof(float)) : 0;
  return w;
}

template <int kDim, bool kBf16, bool kE4m3, bool kWeights>
static void attention_launch(const AttentionArgs& a, const AttentionShape& s, bool row_runs, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(s.workgroups)), block(kWaves * kWave);
  const size_t lds = (kWaves * a.tile_heads * (kDim + 4) + 2 * kWaves * kHeadTile) * sizeof(float);
  if (row_runs) hipLaunchKernelGGL((attention_decode_kernel<kDim, kBf16, kE4m3, true, kWeights>), grid, block, lds, st, a);
  else hipLaunchKernelGGL((attention_decode_kernel<kDim, kBf16, kE4m3, false, kWeights>), grid, block, lds, st, a);
  // few sequences are cut into many pieces each, many into a few
  const int64_t units = static_cast<int64_t>(a.c.batch) * a.q_heads * (kDim / 32);
  const int64_t pieces = a.workgroups / (static_cast<int64_t>(a.c.batch) * a.c.kv_heads * a.head_tiles);
  const dim3 each(static_cast<unsigned>(units)), fourth(static_cast<unsigned>((units + 3) / 4));
  if constexpr (kWeights) {
    if (own_weights(a)) return;
    const float shift = weight_shift(kBf16, kE4m3);
    const size_t stats = (1 + kWaves) * a.group * sizeof(float2);
    const dim3 many(grid.x + each.x), few(grid.x + (s.line ? fourth.x : 0));
    if (s.line && pieces >= kJoinMany)
      hipLaunchKernelGGL((attention_weights_kernel<kDim, kBf16, 16>), many, block, stats, st, a, shift);
    else if (s.line && pieces >= kJoinSome)
      hipLaunchKernelGGL((attention_weights_kernel<kDim, kBf16, 4>), many, block, stats, st, a, shift);
    else
      hipLaunchKernelGGL((attention_weights_kernel<kDim, kBf16, 1>), few, block, stats, st, a, shift);
    return;
  }
  if (!s.line) return;
  if (pieces >= kJoinMany) hipLaunchKernelGGL((attention_join_kernel<kDim, kBf16, 16>), each, dim3(1024), 0, st, a);
  else if (pieces >= kJoinSome) hipLaunchKernelGGL((attention_join_kernel<kDim, kBf16, 4>), each, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((attention_join_kernel<kDim, kBf16, 1>), fourth, dim3(256), 0, st, a);
}

template <int kDim, bool kWeights>
static void attention_by_type(const AttentionArgs& a, const AttentionShape& s, bool bf16, bool row_runs, hipStream_t st) {
  if (a.c.dtype == TRIS_DTYPE_E4M3) {
    if (bf16) attention_launch<kDim, true, true, kWeights>(a, s, row_runs, st);
    else attention_launch<kDim, false, true, kWeights>(a, s, row_runs, st);
  } else {
    if (bf16) attention_launch<kDim, true, false, kWeights>(a, s, row_runs, st);
    else attention_launch<kDim, false, false, kWeights>(a, s, row_runs, st);
  }
}

template <bool kWeights>
static void attention_by_dim(const AttentionArgs& a, const AttentionShape& s, bool bf16, bool row_runs, hipStream_t st) {
  if (a.c.head_dim == 64) attention_by_type<64, kWeights>(a, s, bf16, row_runs, st);
  else if (a.c.head_dim == 128) attention_by_type<128, kWeights>(a, s, bf16, row_runs, st);
  else attention_by_type<256, kWeights>(a, s, bf16, row_runs, st);
}

// What the weights' sums need behind the workspace of the attention alone, in bytes from its beginning; -1: more than 2^62.
struct WeightsSpace {
  int64_t whole_ml, scores, score_row, bytes;
};

static WeightsSpace weights_space(const AttentionSpace& a, int64_t batch, int64_t q_heads, int64_t positions) {
  const auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
  WeightsSpace w;
  w.score_row = (positions + kTileKeys - 1) / kTileKeys * kTileKeys;
  w.whole_ml = up(a.bytes);
  w.scores = w.whole_ml + up(batch * q_heads * static_cast<int64_t>(sizeof(float2)));
  const __int128 end = static_cast<__int128>(batch) * q_heads * w.score_row * static_cast<int64_t>(sizeof(float)) + w.scores;
  w.bytes = end < (static_cast<__int128>(1) << 62) ? static_cast<int64_t>(end) : -1;
  return w;
}

// Query heads of a kv head that the weights' sums take: their statistics are in LDS.
constexpr int kMostGroup = 1024;

// Where the weights are summed.
struct WeightSums {
  float* sums;
  int64_t seq_stride, head_stride;
};

static int attention_decode(const char* who, const void* q, int64_t q_seq_stride, int64_t q_head_stride, int32_t q_type,
                            int32_t q_heads, const tris_paged_cache* cache, float scale, int32_t window, void* out,
                            int64_t out_seq_stride, int64_t out_head_stride, const WeightSums* weights, void* workspace,
                            int64_t workspace_bytes, void* stream) {
  if (const int rc = check_paged_cache(who, cache, q_type)) return rc;
  TRIS_REQUIRE(q_heads >= 1 && q_heads % cache->kv_heads == 0, "%s: q_heads must be a multiple of kv_heads", who);
  TRIS_REQUIRE(window >= 0, "%s: negative window", who);
  if (cache->batch == 0) return TRIS_OK;
  TRIS_REQUIRE(q && out, "%s: null pointer", who);
  for (const int64_t s : {q_seq_stride, q_head_stride, out_seq_stride, out_head_stride})
    TRIS_REQUIRE(s >= 0 && s % 8 == 0, "%s: rows must be 16-byte aligned", who);
  TRIS_REQUIRE(aligned16(q) && aligned16(out), "%s: rows must be 16-byte aligned", who);
  TRIS_REQUIRE(rows_apart<2>({{{cache->batch, out_seq_stride}, {q_heads, out_head_stride}}}, cache->head_dim),
               "%s: output rows overlap", who);
  if (weights) {
    TRIS_REQUIRE(weights->sums || cache->max_pages == 0, "%s: null pointer", who);
    TRIS_REQUIRE(sum_rows_apart(*cache, weights->seq_stride, weights->head_stride), "%s: rows of weight_sum overlap", who);
    TRIS_REQUIRE(q_heads / cache->kv_heads <= kMostGroup, "%s: more than %d query heads for a kv head", who, kMostGroup);
  }
  const int64_t rows = static_cast<int64_t>(cache->batch) * q_heads;
  const AttentionShape s =
      attention_shape(cache->batch, q_heads, cache->kv_heads, cache->head_dim, cache_positions(*cache));
  // a launch has less than 2^32 threads
  TRIS_REQUIRE(rows * (cache->head_dim / 32) < (1LL << 32) / kWave - 4 - (weights && s.line ? 4LL * s.workgroups : 0) &&
                   s.workgroups < (1LL << 32) / (kWaves * kWave),
               "%s: too many rows", who);
  TRIS_REQUIRE(s.places < (1LL << 31) - (1 << 16), "%s: too many positions", who);
  const AttentionSpace w = attention_space(s, cache->batch, cache->kv_heads, cache->head_dim);
  const WeightsSpace ww = weights_space(w, cache->batch, q_heads, cache_positions(*cache));
  const int64_t need = weights ? ww.bytes : w.bytes;
  TRIS_REQUIRE(need >= 0, "%s: too many positions", who);
  TRIS_REQUIRE(need == 0 || (workspace && aligned16(workspace) && workspace_bytes >= need),
               "%s: workspace of %lld bytes needed", who, static_cast<long long>(need));
  AttentionArgs a{static_cast<const uint16_t*>(q),
                  static_cast<uint16_t*>(out),
                  q_seq_stride,
                  q_head_stride,
                  out_seq_stride,
                  out_head_stride,
                  scale * 1.44269504088896341f,
                  window,
                  q_heads,
                  s.group,
                  s.head_tiles,
                  s.tile_heads,
                  s.workgroups,
                  PageDivision(cache->page_size),
                  nullptr,
                  nullptr,
                  nullptr,
                  *cache,
                  nullptr,
                  0,
                  nullptr,
                  nullptr,
                  0,
                  0,
                  0};
  char* at = static_cast<char*>(workspace);
  if (s.line) {
    a.owners = reinterpret_cast<int2*>(at);
    a.part_ml = reinterpret_cast<float2*>(at + w.ml);
    a.part_o = reinterpret_cast<float*>(at + w.o);
  }
  if (weights) {
    a.scores = reinterpret_cast<float*>(at + ww.scores);
    a.score_row = ww.score_row;
    a.whole_ml = reinterpret_cast<float2*>(at + ww.whole_ml);
    a.weight_sum = weights->sums;
    a.sum_seq = weights->seq_stride;
    a.sum_head = weights->head_stride;
    a.sums4 = aligned16(a.weight_sum) && a.sum_seq % 4 == 0 && a.sum_head % 4 == 0;
  }
  bool row_runs = cache->page_size % 16 == 0;
  if (cache->dtype == TRIS_DTYPE_E4M3) {  // four scales a load
    row_runs = row_runs && cache->k_scale_slot_stride == 1 && cache->v_scale_slot_stride == 1 && aligned16(cache->k_scale) &&
            aligned16(cache->v_scale);
    for (const int64_t t : {cache->k_scale_page_stride, cache->k_scale_head_stride, cache->v_scale_page_stride,
                            cache->v_scale_head_stride})
      row_runs = row_runs && t % 4 == 0;
  }
  const bool bf16 = q_type == TRIS_DTYPE_BF16;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (weights) attention_by_dim<true>(a, s, bf16, row_runs, st);
  else attention_by_dim<false>(a, s, bf16, row_runs, st);
  return check_launch(who);
}

}  // namespace tris

using namespace tris;

extern "C" int64_t tris_paged_attention_workspace_bytes(int32_t batch, int32_t q_heads, int32_t kv_heads,
                                                        int32_t head_dim, int32_t max_pages, int32_t page_size) {
  if (batch < 1 || kv_heads < 1 || q_heads < kv_heads || head_dim < 1 || max_pages < 0 || page_size < 1) return 0;
  const int64_t positions = static_cast<int64_t>(max_pages) * page_size;
  return attention_space(attention_shape(batch, q_heads, kv_heads, head_dim, positions), batch, kv_heads, head_dim).bytes;
}

extern "C" int tris_paged_attention_decode(const void* q, int64_t q_seq_stride, int64_t q_head_stride, int32_t q_type,
                                           int32_t q_heads, const tris_paged_cache* cache, float scale, int32_t window,
                                           void* out, int64_t out_seq_stride, int64_t out_head_stride, void* workspace,
                                           int64_t workspace_bytes, void* stream) {
  return attention_decode("tris_paged_attention_decode", q, q_seq_stride, q_head_stride, q_type, q_heads, cache, scale,
                          window, out, out_seq_stride, out_head_stride, nullptr, workspace, workspace_bytes, stream);
}

extern "C" int64_t tris_paged_attention_weights_workspace_bytes(int32_t batch, int32_t q_heads, int32_t kv_heads,
                                                                int32_t head_dim, int32_t max_pages,
                                                                int32_t page_size) {
  if (batch < 1 || kv_heads < 1 || q_heads < kv_heads || head_dim < 1 || max_pages < 0 || page_size < 1) return 0;
  const int64_t positions = static_cast<int64_t>(max_pages) * page_size;
  const AttentionShape s = attention_shape(batch, q_heads, kv_heads, head_dim, positions);
  return weights_space(attention_space(s, batch, kv_heads, head_dim), batch, q_heads, positions).bytes;
}

extern "C" int tris_paged_attention_decode_weights(const void* q, int64_t q_seq_stride, int64_t q_head_stride,
                                                   int32_t q_type, int32_t q_heads, const tris_paged_cache* cache,
                                                   float scale, int32_t window, void* out, int64_t out_seq_stride,
                                                   int64_t out_head_stride, float* weight_sum, int64_t sum_seq_stride,
                                                   int64_t sum_head_stride, void* workspace, int64_t workspace_bytes,
                                                   void* stream) {
  const WeightSums weights{weight_sum, sum_seq_stride, sum_head_stride};
  return attention_decode("tris_paged_attention_decode_weights", q, q_seq_stride, q_head_stride, q_type, q_heads, cache,
                          scale, window, out, out_seq_stride, out_head_stride, &weights, workspace, workspace_bytes, stream);
}
