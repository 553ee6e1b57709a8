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
// No operand goes through LDS, the statistics of a head stay in its lanes, and rescaling is a product in a lane.
//
// The work is split over the length: every wavefront of the grid derives the same plan from seq_lens (the total of
// tiles, a chunk per workgroup, the workgroups of each sequence), so the launch needs no lengths on the host and a long
// sequence beside short ones gets its share of the GPU.  A sequence in one piece is written at once, the pieces of a
// longer one leave fp32 sums in the workspace, and a second launch joins them.
#include <algorithm>

#include "tris_paged.h"

namespace tris {

constexpr int kTileKeys = 32;
constexpr int kWaves = 4;          // wavefronts of a workgroup, taking its tiles in turn
constexpr int kHeadTile = 16;      // query heads of a workgroup
constexpr int kTargetWorkgroups = 1024;

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
  int32_t window, q_heads, group, head_tiles, tile_heads, max_slots;
  PageDivision page_of;
  int2* plan;                        // [batch]: first slot and number of the sequence's pieces
  float2* part_ml;                   // [slots][kv_heads * head_tiles][tile_heads]: maximum and sum
  float* part_o;                     // the same rows of head_dim sums
  tris_paged_cache c;
};

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// the positions [first, n) that sequence b's token attends to
__device__ __forceinline__ void sequence_range(const AttentionArgs& a, int b, int* n, int* first) {
  *n = b < a.c.batch ? min(max(a.c.seq_lens[b], 0), cache_positions(a.c)) : 0;
  *first = a.window > 0 ? max(0, *n - a.window) : 0;
}
__device__ __forceinline__ int range_tiles(int n, int first) {
  return n > first ? (n + kTileKeys - 1) / kTileKeys - first / kTileKeys : 0;
}

struct Piece {
  int b, n, first, t0, t1, splits, slot;  // slot: of this piece; only sequences in several pieces have slots
};

// Piece `item` of the plan (the same for every caller): with T tiles in all, a workgroup gets
// chunk = max(4, T * head groups / kTargetWorkgroups) tiles rounded up to one for each wavefront, and sequence b is cut
// into ceil(tiles / chunk) pieces, an idle one into one of no tiles.  At most kTargetWorkgroups / head groups + batch
// pieces come of it.
__device__ __forceinline__ bool find_piece(const AttentionArgs& a, int item, int head_groups, Piece* p) {
  const int lane = threadIdx.x % kWave;
  int n, first;
  float total = 0.0f;
  for (int b0 = 0; b0 < a.c.batch; b0 += kWave) {
    sequence_range(a, b0 + lane, &n, &first);
    total += wave_sum_f32(static_cast<float>(range_tiles(n, first)));
  }
  const float share = fminf(total * static_cast<float>(head_groups) / static_cast<float>(kTargetWorkgroups), 1e9f);
  const int chunk = max(1, (static_cast<int>(ceilf(share)) + kWaves - 1) / kWaves) * kWaves;
  int pieces = 0, slots = 0;
  for (int b0 = 0; b0 < a.c.batch; b0 += kWave) {
    const int b = b0 + lane;
    sequence_range(a, b, &n, &first);
    const int tiles = range_tiles(n, first);
    const int s = b < a.c.batch ? max(1, (tiles + chunk - 1) / chunk) : 0;
    const int end = pieces + wave_incl_sum_i32(s);
    const int slot_end = slots + wave_incl_sum_i32(s > 1 ? s : 0);
    const uint64_t hit = __ballot(item >= end - s && item < end);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      const int at = item - __builtin_amdgcn_readlane(end - s, l);
      p->b = b0 + l;
      p->n = __builtin_amdgcn_readlane(n, l);
      p->first = __builtin_amdgcn_readlane(first, l);
      p->splits = __builtin_amdgcn_readlane(s, l);
      p->slot = __builtin_amdgcn_readlane(slot_end, l) - p->splits + at;
      p->t0 = p->first / kTileKeys + at * chunk;
      p->t1 = min(p->first / kTileKeys + __builtin_amdgcn_readlane(tiles, l), p->t0 + chunk);
      return true;
    }
    pieces = __builtin_amdgcn_readlane(end, kWave - 1);
    slots = __builtin_amdgcn_readlane(slot_end, kWave - 1);
  }
  return false;
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

// kWhole: every 16 keys of a tile lie in one page (page_size a multiple of 16; with e4m3, scale rows that can be read
// four at a time), so that page numbers and row addresses are the same for the whole wavefront; else each lane looks
// up the pages of its own keys.
template <int kDim, bool kBf16, bool kE4m3, bool kWhole>
__global__ __launch_bounds__(kWaves * kWave, kDim == 256 ? 1 : 2) void attention_decode_kernel(const AttentionArgs a) {
  constexpr bool kBf16V = kBf16 || kE4m3;           // type of the value product (see the probabilities below)
  constexpr int kRun = kDim < 128 ? kDim / 16 : 8;  // dimensions of one of a lane's runs of a value row
  constexpr int kRuns = kDim / 16 / kRun;
  constexpr int kSize = kE4m3 ? 1 : 2;
  constexpr int kKLoads = kDim * kSize / 64;        // 16-byte loads of a lane for one key row's quarter
  constexpr int kVWords = kRun * kSize / 4;         // words of a run
  constexpr int kPad = kDim + 4;
  extern __shared__ float lds[];                    // [kWaves][tile_heads][kPad] sums, then [kWaves][16] factors and sums

  const int head_groups = a.c.kv_heads * a.head_tiles;
  const int hg = static_cast<int>(blockIdx.x) % head_groups;
  Piece p;
  if (!find_piece(a, static_cast<int>(blockIdx.x) / head_groups, head_groups, &p)) return;
  const int b = uniform(p.b), n = uniform(p.n), first = uniform(p.first);
  const int kvh = hg / a.head_tiles, head0 = (hg % a.head_tiles) * kHeadTile;
  const int heads = min(kHeadTile, a.group - head0);
  const int wave = uniform(threadIdx.x / kWave), lane = threadIdx.x % kWave, col = lane % 16, g = lane / 16;

  // the query operand: head col, the dimensions that the K operand's lane has
  u32x4 q[kDim / 32];
#pragma unroll
  for (int i = 0; i < kDim / 32; ++i) {
    const int d = kE4m3 ? (i / 2) * 64 + g * 16 + (i % 2) * 8 : i * 32 + g * 8;
    q[i] = u32x4{0, 0, 0, 0};
    if (col < heads)
      q[i] = *reinterpret_cast<const u32x4*>(a.q + b * a.q_seq + (kvh * a.group + head0 + col) * a.q_head + d);
  }

  const char* kbase = static_cast<const char*>(a.c.k) + kvh * a.c.k_head_stride * kSize;
  const char* vbase = static_cast<const char*>(a.c.v) + kvh * a.c.v_head_stride * kSize;
  const float* ksbase = kE4m3 ? a.c.k_scale + kvh * a.c.k_scale_head_stride : nullptr;
  const float* vsbase = kE4m3 ? a.c.v_scale + kvh * a.c.v_scale_head_stride : nullptr;
  const int32_t* table = a.c.block_table + b * a.c.table_stride;
  const int k_slot = static_cast<int>(a.c.k_slot_stride) * kSize, v_slot = static_cast<int>(a.c.v_slot_stride) * kSize;
  const int ks_slot = static_cast<int>(a.c.k_scale_slot_stride), vs_slot = static_cast<int>(a.c.v_scale_slot_stride);

  // the pages of a tile's keys, -1 where there is none: of its two halves, or of the lane's two key rows and eight
  // value rows
  constexpr int kPages = kWhole ? 2 : 10;
  struct Pages { int id[kPages]; };
  const auto key_of = [&](int tile, int i) {
    if constexpr (kWhole) return tile * kTileKeys + i * 16;
    else if (i < 2) return tile * kTileKeys + i * 16 + col;
    else return tile * kTileKeys + ((i - 2) / 4) * 16 + g * 4 + (i - 2) % 4;
  };
  const auto find_pages = [&](int tile) {
    Pages pg;
#pragma unroll
    for (int i = 0; i < kPages; ++i) {
      const int key = key_of(tile, i);
      int id = -1;
      if (tile < p.t1 && key < n && (kWhole || key >= first)) id = table[a.page_of(key)];
      pg.id[i] = static_cast<uint32_t>(id) < static_cast<uint32_t>(a.c.num_pages) ? id : -1;
      if constexpr (kWhole) pg.id[i] = uniform(pg.id[i]);
    }
    return pg;
  };

  u32x4 kr[2][kKLoads];
  uint32_t vr[8][kRuns * kVWords];
  float ks[8], vs[8];
  // rows without a page read page 0; their keys are masked
  const auto load_k = [&](int tile, const Pages& pg) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int page = max(pg.id[t], 0), key = key_of(tile, t);
      const int slot = key - a.page_of(key) * a.c.page_size;
      const char* row = kbase + page * a.c.k_page_stride * kSize;
      uint32_t off;
      if constexpr (kWhole) {
        row += static_cast<int64_t>(slot) * k_slot;
        off = static_cast<uint32_t>(col * k_slot + g * 16);
      } else {
        off = static_cast<uint32_t>(slot * k_slot + g * 16);
      }
#pragma unroll
      for (int i = 0; i < kKLoads; ++i) kr[t][i] = *reinterpret_cast<const u32x4*>(row + off + i * 64);
      if constexpr (kE4m3 && kWhole) {
        const f32x4 s = *reinterpret_cast<const f32x4*>(ksbase + page * a.c.k_scale_page_stride + slot + g * 4);
#pragma unroll
        for (int r = 0; r < 4; ++r) ks[t * 4 + r] = s[r];
      }
    }
    if constexpr (kE4m3 && !kWhole) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int key = key_of(tile, 2 + j), slot = key - a.page_of(key) * a.c.page_size;
        ks[j] = ksbase[max(pg.id[2 + j], 0) * a.c.k_scale_page_stride + slot * ks_slot];
      }
    }
  };
  const auto load_v = [&](int tile, const Pages& pg) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = kWhole ? j / 4 : 2 + j;
      const int page = max(pg.id[i], 0), key = key_of(tile, i);
      const int slot = key - a.page_of(key) * a.c.page_size;
      const char* row = vbase + page * a.c.v_page_stride * kSize;
      uint32_t off;
      if constexpr (kWhole) {
        row += static_cast<int64_t>(slot) * v_slot;
        off = static_cast<uint32_t>((g * 4 + j % 4) * v_slot + col * kRun * kSize);
      } else {
        off = static_cast<uint32_t>(slot * v_slot + col * kRun * kSize);
        if constexpr (kE4m3) vs[j] = vsbase[page * a.c.v_scale_page_stride + slot * vs_slot];
      }
#pragma unroll
      for (int c = 0; c < kRuns; ++c) {
        const char* src = row + off + c * 16 * kRun * kSize;
        uint32_t* dst = vr[j] + c * kVWords;
        if constexpr (kVWords == 4) *reinterpret_cast<u32x4*>(dst) = *reinterpret_cast<const u32x4*>(src);
        else if constexpr (kVWords == 2) *reinterpret_cast<u32x2*>(dst) = *reinterpret_cast<const u32x2*>(src);
        else *dst = *reinterpret_cast<const uint32_t*>(src);
      }
      if constexpr (kE4m3 && kWhole) {
        if (j % 4 == 0) {
          const f32x4 s = *reinterpret_cast<const f32x4*>(vsbase + page * a.c.v_scale_page_stride + slot + g * 4);
#pragma unroll
          for (int r = 0; r < 4; ++r) vs[j + r] = s[r];
        }
      }
    }
  };

  float m = -INFINITY, l = 0.0f;
  f32x4 acc[kRuns * kRun];
#pragma unroll
  for (int i = 0; i < kRuns * kRun; ++i) acc[i] = f32x4{0, 0, 0, 0};

  int tile = uniform(p.t0) + wave;
  const int t1 = uniform(p.t1);
  Pages cur = find_pages(tile), nxt = find_pages(tile + kWaves);
  if (tile < t1) {
    load_k(tile, cur);
    load_v(tile, cur);
  }
  for (; tile < t1; tile += kWaves) {
    const bool more = tile + kWaves < t1;
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
        s[t] = mfma<kBf16>(k, q[i], s[t]);
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
    if constexpr (kWhole) {
      edge = edge || cur.id[0] < 0 || cur.id[1] < 0;
    } else {
      bool hole = false;
#pragma unroll
      for (int j = 0; j < 8; ++j) hole = hole || cur.id[2 + j] < 0;
      edge = __any(hole);
    }
    bool valid[8];
    if (edge) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int key = key0 + (j / 4) * 16 + g * 4 + j % 4;
        valid[j] = key >= first && key < n && cur.id[kWhole ? j / 4 : 2 + j] >= 0;
        x[j] = valid[j] ? x[j] : -INFINITY;
      }
    }
    if (more) load_k(tile + kWaves, nxt);

    float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
    if (__any(top > m)) {
      const float now = across_groups(fmaxf(m, top), [](float u, float w) { return fmaxf(u, w); });
      const float f = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - now);
      m = now;
      l *= f;
#pragma unroll
      for (int i = 0; i < kRuns * kRun; ++i) acc[i] *= f;
    }
    // The probabilities enter the value product as two 16-bit parts, the value and what its rounding left, so that the
    // result has one rounding to speak of, the output's.  In fp16 they are 2^15 times as large (the sum too, so that it
    // cancels): a long tail far below the maximum would lose its bits to the subnormals otherwise.  An 8-bit cache's
    // product runs in bf16, whose range takes any scale; its elements are exact in either type.
    const float base = (m == -INFINITY ? 0.0f : m) - (kBf16V ? 0.0f : 15.0f);
    float w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      w[j] = __builtin_amdgcn_exp2f(x[j] - base);
      l += w[j];
      if constexpr (kE4m3) w[j] *= vs[j];
    }
    if (edge) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        w[j] = valid[j] ? w[j] : 0.0f;
#pragma unroll
        for (int i = 0; i < kRuns * kVWords; ++i) vr[j][i] = valid[j] ? vr[j][i] : 0u;
      }
    }
    u32x4 hi, lo;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float w0 = w[2 * i], w1 = w[2 * i + 1];
      if constexpr (kBf16V) {
        const uint32_t u0 = __float_as_uint(w0), u1 = __float_as_uint(w1);
        hi[i] = __builtin_amdgcn_perm(u1, u0, 0x07060302u);
        lo[i] = pack_bf16_rne(w0 - __uint_as_float(u0 & 0xFFFF0000u), w1 - __uint_as_float(u1 & 0xFFFF0000u));
      } else {
        const auto h = __builtin_amdgcn_cvt_pkrtz(w0, w1);
        hi[i] = __builtin_bit_cast(uint32_t, h);
        lo[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(w0 - static_cast<float>(h[0]), w1 - static_cast<float>(h[1])));
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
          o = mfma<kBf16V>(v, hi, o);
          o = mfma<kBf16V>(v, lo, o);
        }
      }
    }
    if (more) load_v(tile + kWaves, nxt);
    cur = nxt;
    nxt = find_pages(tile + 2 * kWaves);
  }

  // the wavefronts' sums joined under the workgroup's maximum
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
  const int64_t row0 = (static_cast<int64_t>(p.slot) * head_groups + hg) * a.tile_heads;
  for (int i = threadIdx.x * 2; i < heads * kDim; i += kWaves * kWave * 2) {
    const int h = i / kDim, d = i % kDim;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, sh_m[w * kHeadTile + h]);
    const float base = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f, y0 = 0.0f, y1 = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = __builtin_amdgcn_exp2f(sh_m[w * kHeadTile + h] - base);
      const float* o = sh_o + (w * a.tile_heads + h) * kPad + d;
      sum += sh_l[w * kHeadTile + h] * f;
      y0 += o[0] * f;
      y1 += o[1] * f;
    }
    if (p.splits == 1) {
      const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
      uint16_t* dst = a.out + b * a.out_seq + (kvh * a.group + head0 + h) * a.out_head + d;
      *reinterpret_cast<uint32_t*>(dst) = kBf16 ? pack_bf16_rne(y0 * f, y1 * f) : pack_f16_rne(y0 * f, y1 * f);
    } else if (p.slot < a.max_slots) {
      *reinterpret_cast<float2*>(a.part_o + (row0 + h) * kDim + d) = make_float2(y0, y1);
      if (d == 0) a.part_ml[row0 + h] = make_float2(top, sum);
    }
  }
  if (a.plan != nullptr && hg == 0 && threadIdx.x == 0 && p.t0 == p.first / kTileKeys)
    a.plan[b] = make_int2(p.splits > 1 ? p.slot : 0, p.splits);
}

// Joins the pieces of one (sequence, query head): the maximum over them, then each wavefront adds every fourth piece.
template <int kDim, bool kBf16>
__global__ __launch_bounds__(kWaves * kWave) void attention_join_kernel(const AttentionArgs a) {
  constexpr int kPer = kDim / kWave;
  __shared__ float sh_l[kWaves], sh_o[kWaves][kDim];
  const int b = static_cast<int>(blockIdx.x) / a.q_heads, h = static_cast<int>(blockIdx.x) % a.q_heads;
  const int2 plan = a.plan[b];
  if (plan.y <= 1) return;
  const int kvh = h / a.group, in = h % a.group, head_groups = a.c.kv_heads * a.head_tiles;
  const int hg = kvh * a.head_tiles + in / kHeadTile;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const int pieces = min(plan.y, a.max_slots - plan.x);
  const auto row = [&](int i) {
    return (static_cast<int64_t>(plan.x + i) * head_groups + hg) * a.tile_heads + in % kHeadTile;
  };
  float top = -INFINITY;
  for (int i = lane; i < pieces; i += kWave) top = fmaxf(top, a.part_ml[row(i)].x);
  top = wave_max_f32(top);
  const float base = top == -INFINITY ? 0.0f : top;
  float l = 0.0f, o[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) o[e] = 0.0f;
#pragma unroll 4
  for (int i = wave; i < pieces; i += kWaves) {
    const int64_t r = row(i);
    const float2 ml = a.part_ml[r];
    const float f = __builtin_amdgcn_exp2f(ml.x - base);
    l += ml.y * f;
#pragma unroll
    for (int e = 0; e < kPer; ++e) o[e] += a.part_o[r * kDim + lane * kPer + e] * f;
  }
  if (lane == 0) sh_l[wave] = l;
#pragma unroll
  for (int e = 0; e < kPer; ++e) sh_o[wave][lane * kPer + e] = o[e];
  __syncthreads();
  const float sum = ((sh_l[0] + sh_l[1]) + sh_l[2]) + sh_l[3];
  const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
  for (int d = threadIdx.x; d < kDim; d += kWaves * kWave) {
    const float y = (((sh_o[0][d] + sh_o[1][d]) + sh_o[2][d]) + sh_o[3][d]) * f;
    store1(a.out, b * a.out_seq + h * a.out_head + d, y, kBf16 ? TRIS_DTYPE_BF16 : TRIS_DTYPE_F16);
  }
}

// The launch's sizes, from shapes alone.
struct AttentionShape {
  int group, head_tiles, tile_heads, head_groups;
  int64_t pieces, slots;  // bounds of the plan
  bool splits;            // whether any sequence can be cut
};

static AttentionShape attention_shape(int64_t batch, int q_heads, int kv_heads, int64_t positions) {
  AttentionShape s;
  s.group = q_heads / kv_heads;
  s.head_tiles = (s.group + kHeadTile - 1) / kHeadTile;
  s.tile_heads = s.group < kHeadTile ? s.group : kHeadTile;
  s.head_groups = kv_heads * s.head_tiles;
  // tiles of a sequence (a window may add one by its start inside a tile), pieces of at least kWaves tiles
  const int64_t tiles = positions / kTileKeys + 2;
  const int64_t most = (tiles + kWaves - 1) / kWaves;
  const int64_t shared = kTargetWorkgroups / s.head_groups + 1;
  s.pieces = std::min(batch * most, shared + batch);
  // pieces of sequences that are cut: each such sequence has at most twice tiles / chunk
  s.slots = std::min(batch * most, 2 * shared);
  s.splits = most > 1;
  return s;
}

struct AttentionSpace {
  int64_t ml, o, bytes;
};

static AttentionSpace attention_space(const AttentionShape& s, int64_t batch, int head_dim) {
  const auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
  AttentionSpace w;
  const int64_t rows = s.slots * s.head_groups * s.tile_heads;
  w.ml = up(batch * static_cast<int64_t>(sizeof(int2)));
  w.o = w.ml + up(rows * static_cast<int64_t>(sizeof(float2)));
  w.bytes = s.splits ? w.o + rows * head_dim * static_cast<int64_t>(sizeof(float)) : 0;
  return w;
}

template <int kDim, bool kBf16, bool kE4m3>
static void attention_launch(const AttentionArgs& a, const AttentionShape& s, bool whole, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(s.pieces * s.head_groups)), block(kWaves * kWave);
  const size_t lds = (kWaves * a.tile_heads * (kDim + 4) + 2 * kWaves * kHeadTile) * sizeof(float);
  if (whole) hipLaunchKernelGGL((attention_decode_kernel<kDim, kBf16, kE4m3, true>), grid, block, lds, st, a);
  else hipLaunchKernelGGL((attention_decode_kernel<kDim, kBf16, kE4m3, false>), grid, block, lds, st, a);
  if (s.splits)
    hipLaunchKernelGGL((attention_join_kernel<kDim, kBf16>), dim3(static_cast<unsigned>(a.c.batch * a.q_heads)), block,
                       0, st, a);
}

template <int kDim>
static void attention_by_type(const AttentionArgs& a, const AttentionShape& s, bool bf16, bool whole, hipStream_t st) {
  if (a.c.dtype == TRIS_DTYPE_E4M3) {
    if (bf16) attention_launch<kDim, true, true>(a, s, whole, st);
    else attention_launch<kDim, false, true>(a, s, whole, st);
  } else {
    if (bf16) attention_launch<kDim, true, false>(a, s, whole, st);
    else attention_launch<kDim, false, false>(a, s, whole, st);
  }
}

}  // namespace tris

using namespace tris;

extern "C" int64_t tris_paged_attention_workspace_bytes(int32_t batch, int32_t q_heads, int32_t kv_heads,
                                                        int32_t head_dim, int32_t max_pages, int32_t page_size) {
  if (batch < 1 || kv_heads < 1 || q_heads < kv_heads || head_dim < 1 || max_pages < 0 || page_size < 1) return 0;
  return attention_space(attention_shape(batch, q_heads, kv_heads, static_cast<int64_t>(max_pages) * page_size), batch,
                         head_dim).bytes;
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
  const int64_t rows = static_cast<int64_t>(cache->batch) * q_heads;
  const AttentionShape s = attention_shape(cache->batch, q_heads, cache->kv_heads, cache_positions(*cache));
  TRIS_REQUIRE(rows <= 2147483647LL && s.pieces * s.head_groups <= 2147483647LL, "%s: too many rows", who);
  const AttentionSpace w = attention_space(s, cache->batch, cache->head_dim);
  TRIS_REQUIRE(w.bytes == 0 || (workspace && aligned16(workspace) && workspace_bytes >= w.bytes),
               "%s: workspace of %lld bytes needed", who, static_cast<long long>(w.bytes));
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
                  0,
                  PageDivision(cache->page_size),
                  nullptr,
                  nullptr,
                  nullptr,
                  *cache};
  if (s.splits) {
    char* at = static_cast<char*>(workspace);
    a.max_slots = static_cast<int32_t>(s.slots);
    a.plan = reinterpret_cast<int2*>(at);
    a.part_ml = reinterpret_cast<float2*>(at + w.ml);
    a.part_o = reinterpret_cast<float*>(at + w.o);
  }
  bool whole = cache->page_size % 16 == 0;
  if (cache->dtype == TRIS_DTYPE_E4M3) {  // four scales a load
    whole = whole && cache->k_scale_slot_stride == 1 && cache->v_scale_slot_stride == 1 && aligned16(cache->k_scale) &&
            aligned16(cache->v_scale);
    for (const int64_t t : {cache->k_scale_page_stride, cache->k_scale_head_stride, cache->v_scale_page_stride,
                            cache->v_scale_head_stride})
      whole = whole && t % 4 == 0;
  }
  const bool bf16 = q_type == TRIS_DTYPE_BF16;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (cache->head_dim == 64) attention_by_type<64>(a, s, bf16, whole, st);
  else if (cache->head_dim == 128) attention_by_type<128>(a, s, bf16, whole, st);
  else attention_by_type<256>(a, s, bf16, whole, st);
  return check_launch(who);
}
