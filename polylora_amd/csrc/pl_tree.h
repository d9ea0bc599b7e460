// What the two kernels of pl_tree_attention share: arguments, what of a row counts, and
// how the batch's work is dealt out.
#pragma once

#include <type_traits>

#include "pl_attend.h"

struct tree_args {
  const void* q;
  int64_t q_row, q_token, q_head;
  pl_cache_view key, value;
  pl_page_table table;
  const int32_t *past, *seq_lens;
  const int32_t* visible;  // [rows][tokens][words], null: a token sees those before it
  int64_t visible_row, visible_token;
  const int32_t* depths;
  int64_t depths_row;
  const float *k_scale, *v_scale;
  void* out;  // contiguous [rows][row_len][heads][dim]
  float* parts;
  int32_t* counters;
  float scale;
  int32_t rows, row_len, heads, kv_heads, dim, window, group;
  int32_t tok0, toks;           // the tokens of this launch
  int32_t col_tiles, slices;    // workers: col_tiles for each slice
  float per_group;              // 1 / group
  int32_t once;                 // keys and values are read once and stay in no cache
};

namespace {

constexpr int kCus = 256;
constexpr int kWorkersMax = 2 * kCus;

// Parts of 16 bits that a weight enters its product as: three bf16 hold it whole, two fp16 keep
// 2^-21 of it, as in paged_attention.hip.  Two bf16 keep 17 of its 24 bits, and small differences
// of values come out wrong by percents; the third takes (bf16, 32 query heads over 8 of 128) 64 x 8 drafts over 4096
// tokens 153 -> 155 us, 64 x 16 183 -> 187, 64 x 32 240 -> 267, 16 over 131072 in 8 bits 91 -> 103.
template <int DT>
constexpr int kWeightParts = DT == PL_BF16 ? 3 : 2;
// log2 of how far scores may pass the maximum that weights are taken against, and of
// what fp16 weights are multiplied by, that their parts keep small ones: to 2^15.  (They end
// at 2^-31 of the largest, 2^-39 where the maximum lags by all of it, in their sum as in the output.)
constexpr float kSlack = 8.f;

// A row's tokens that count, for the tokens of this launch.
struct tree_span {
  int first, len, past, n, base, atoms;
};
template <int ATOM>
__device__ __forceinline__ tree_span span_of(const tree_args& a, int past, int n) {
  const int64_t cap = a.table.num_pages ? (int64_t)a.table.max_pages << a.table.page_shift : 0;
  tree_span r;
  r.n = min(n, a.row_len), r.past = past;
  const bool live = r.n > a.tok0 && past >= 0;
  r.len = live ? (int)min((int64_t)past + r.n, cap) : 0;
  const int64_t first = (int64_t)past + (a.visible ? 0 : a.tok0) - a.window + 1;
  // (a window that begins behind the pages' end sees nothing of them)
  r.first = live && a.window > 0 ? (int)min(max(first, (int64_t)0), (int64_t)r.len) : 0;
  r.base = r.first & ~31;
  r.atoms = max(1, (r.len - r.base + ATOM - 1) / ATOM);  // an empty row's output is an atom too
  return r;
}

// Not 0 where a word of values holds an infinity or NaN: an exponent (and, of e4m3, a
// mantissa) of ones carries into the sign's place when one is added at its end.
template <int DT, int CT>
__device__ __forceinline__ uint32_t nonfinite_bits(uint32_t w) {
  if constexpr (CT == PL_F8E4M3)
    return (w & 0x7f7f7f7fu) + 0x01010101u & 0x80808080u;
  else if constexpr (DT == PL_F32)
    return (w & 0x7f800000u) + 0x00800000u & 0x80000000u;
  else if constexpr (DT == PL_BF16)
    return (w & 0x7f807f80u) + 0x00800080u & 0x80008000u;
  else
    return (w & 0x7c007c00u) + 0x04000400u & 0x80008000u;
}
// A word of values without its infinities and NaN.
template <int DT, int CT>
__device__ __forceinline__ uint32_t finite_part(uint32_t w) {
  if constexpr (CT == PL_F8E4M3) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w &= (w >> 8 * i & 0x7f) == 0x7f ? ~(0xffu << 8 * i) : ~0u;
  } else if constexpr (DT == PL_F32) {
    w &= (w & 0x7f800000u) == 0x7f800000u ? 0u : ~0u;
  } else {
    constexpr uint32_t kExp = DT == PL_BF16 ? 0x7f80u : 0x7c00u;
    w &= (w & kExp) == kExp ? 0xffff0000u : ~0u;
    w &= (w & kExp << 16) == kExp << 16 ? 0x0000ffffu : ~0u;
  }
  return w;
}
template <int DT, int CT>
__device__ __forceinline__ float value_element(const uint32_t* w, int i) {
  if constexpr (DT == PL_F32)
    return __uint_as_float(w[i]);
  else if constexpr (CT == PL_F8E4M3)
    return unpack<DT>(i % 4 < 2 ? widen<DT, false>(w[i / 4]) : widen<DT, true>(w[i / 4]), i % 2);
  else
    return unpack<DT>(w[i / 2], i % 2);
}

// Whole pairs or equal runs, from the atoms' number, the pairs and the longest of
// them, in tiles of a wave (paged_attention.hip has the measurements).
constexpr float kFirst = 2.f, kPair = 8.6f, kJoin = 5.f;
template <int TILES>
__device__ __forceinline__ bool choose_whole(int slices, int total, int pairs, int longest) {
  const float w = (float)slices, n = (float)total * TILES, top = (float)longest * TILES;
  const float ends = kFirst * w + kPair * (float)pairs;
  return top * w + n + ends < w + n + ends + kJoin * w;
}

// Workers of one slice of tokens, one for each column tile, run side by side on one
// XCD: the first to ask for a tile brings it into the L2 that the others read.
struct tree_worker {
  int ct, slice;
};
__device__ __forceinline__ tree_worker worker_of(const tree_args& a) {
  const int round = (int)blockIdx.x / kXcds;
  return {round % a.col_tiles, (int)blockIdx.x % kXcds + kXcds * (round / a.col_tiles)};
}
// Workers of a launch: `most` at most, `need` slices at most.
inline int slices_of(int64_t atoms_most, int most, int col_tiles) {
  const int64_t fit = most / (kXcds * col_tiles), need = (atoms_most + kXcds - 1) / kXcds;
  return kXcds * (int)(need < fit ? need : fit > 0 ? fit : 1);
}

// The run of atoms of a slice, and the row of its first.
struct tree_run {
  int from, to, per, total, row, row_start, row_past, row_new;
  bool whole_pairs;
};
template <int ATOM, int TILES>
__device__ __forceinline__ tree_run find_run(const tree_args& a, int slice, int lane, bool one_of_many = false) {
  tree_run r;
  // Each wave works out the deal for itself: 64 rows to a look, no barrier.
  constexpr int kLooks = 2;  // that stay in registers
  int pasts[kLooks], counts[kLooks], atoms[kLooks], total = 0, longest = 0;
#pragma unroll
  for (int k = 0; k < kLooks; ++k) {
    const int b = min(k * 64 + lane, a.rows - 1);
    pasts[k] = a.past[b], counts[k] = a.seq_lens ? a.seq_lens[b] : a.row_len;
  }
#pragma unroll
  for (int k = 0; k < kLooks; ++k) {
    const int n = span_of<ATOM>(a, pasts[k], counts[k]).atoms;
    atoms[k] = k * 64 + lane < a.rows ? n : 0;
    total += atoms[k], longest = max(longest, atoms[k]);
  }
  for (int b = kLooks * 64 + lane; b < a.rows; b += 64) {
    const int n = span_of<ATOM>(a, a.past[b], a.seq_lens ? a.seq_lens[b] : a.row_len).atoms;
    total += n, longest = max(longest, n);
  }
  total = __builtin_amdgcn_readlane(scan_sum(total), 63) * a.kv_heads;
  longest = __builtin_amdgcn_readlane(scan_max(longest), 63);
  // where asked for, one workgroup on a CU for many atoms (see paged_attention.hip)
  const int slices = one_of_many && total >= 8 * kCus ? min(a.slices, kCus) : a.slices;
  const bool whole_pairs = choose_whole<TILES>(slices, total, a.rows * a.kv_heads, longest);
  const int per = (total + slices - 1) / slices;
  r.from = (int)min((int64_t)slice * per, (int64_t)total);
  r.to = min(total - per, r.from) + per;
  r.per = per, r.total = total, r.whole_pairs = whole_pairs;
  r.row = r.row_start = r.row_past = r.row_new = 0;
  if (r.from >= total) return r;
  // the row of its first atom: the first whose atoms up to and with it pass `from`
  for (int b0 = 0;; b0 += 64) {
    const int b = b0 + lane;
    int n = atoms[0], past = pasts[0], count = counts[0];
#pragma unroll
    for (int k = 1; k < kLooks; ++k) {
      n = b0 == k * 64 ? atoms[k] : n;
      past = b0 == k * 64 ? pasts[k] : past;
      count = b0 == k * 64 ? counts[k] : count;
    }
    if (b0 >= kLooks * 64) {
      past = b < a.rows ? a.past[b] : 0;
      count = b < a.rows ? a.seq_lens ? a.seq_lens[b] : a.row_len : 0;
      n = b < a.rows ? span_of<ATOM>(a, past, count).atoms : 0;
    }
    n *= a.kv_heads;
    const int upto = scan_sum(n) + r.row_start;
    const uint64_t passed = __ballot(upto > r.from);
    if (passed || b0 + 64 >= a.rows) {
      const int hit = passed ? __ffsll((long long)passed) - 1 : 63;
      r.row = b0 + hit;
      r.row_start = __builtin_amdgcn_readlane(upto - n, hit);
      r.row_past = __builtin_amdgcn_readlane(past, hit);
      r.row_new = __builtin_amdgcn_readlane(count, hit);
      break;
    }
    r.row_start = __builtin_amdgcn_readlane(upto, 63);
  }
  r.row = uniform(r.row);
  return r;
}

// Token and head of a column of the launch (toks * group of them): a quotient below 2^12
// by way of fp32, half a column away from the next one.
struct column_place {
  int token, head;
};
__device__ __forceinline__ column_place place_of(const tree_args& a, int col, int hk) {
  const int t = (int)(((float)col + 0.5f) * a.per_group);
  return {a.tok0 + t, hk * a.group + col - t * a.group};
}

// The weights of a column's eight tokens of a tile as 16-bit parts, two tokens to a word.
// No part is negative, or 0 beside the first, so that an infinite value stays one.
template <int DT>
__device__ __forceinline__ void weight_parts(const float* p, pl_u32x4* part) {
  constexpr int kParts = kWeightParts<DT>;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float x = p[2 * j], y = p[2 * j + 1];
#pragma unroll
    for (int k = 0; k < kParts; ++k) {
      // bf16's last part is exact either way
      const uint32_t z = k + 1 < kParts || DT == PL_BF16 ? pack2_down<DT>(x, y) : pack2<DT>(x, y);
      x -= unpack<DT>(z, 0), y -= unpack<DT>(z, 1);
      part[k][j] = k ? at_least_smallest<DT>(z, part[0][j]) : z;
    }
  }
}

// Which of four places from `place` on, which all hold tokens or none that count, a column
// of token t (-1: none that counts) sees, which sees places from `first` on: a bit each.
// The mask's words are read whatever they are for, so that a tile's reads are
// on their way together.
__device__ __forceinline__ uint32_t column_sees(const tree_args& a, const tree_span& r, int row, int t, int first,
                                                int place) {
  const int draft = place - r.past;
  uint32_t bits;
  if (a.visible) {
    typedef const __attribute__((address_space(1))) int32_t* global_i32;
    const global_i32 words = (global_i32)(a.visible + row * a.visible_row + max(t, 0) * a.visible_token);
    const int at = min(max(draft, 0), a.row_len - 1) >> 5, after = min(at + 1, (a.row_len - 1) >> 5);
    uint32_t low = (uint32_t)words[at], high = (uint32_t)words[after];
    asm volatile("" : "+v"(low), "+v"(high));
    const uint64_t both = (uint64_t)high << 32 | low;
    // drafts below 0 are the lower places of a four that begins before the drafts
    bits = draft >= 0 ? (uint32_t)(both >> (draft & 31)) : (uint32_t)both << min(-draft, 31);
  } else {
    bits = draft > t ? 0u : 0xfu >> max(0, 3 - (t - draft));
  }
  uint32_t yes = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const bool before = draft + k < 0, late = place + k >= first;
    yes |= (uint32_t)(before ? late : (bits >> k & 1) && (a.visible || late)) << k;
  }
  return t >= 0 ? yes : 0u;
}
// The first place that token t sees (of those before the drafts, in a tree).
__device__ __forceinline__ int first_seen(const tree_args& a, const tree_span& r, int row, int t) {
  if (a.window <= 0 || t < 0) return 0;
  const int depth = a.depths ? max(a.depths[row * a.depths_row + t], 0) : t;
  return (int)min(max((int64_t)r.past + depth - a.window + 1, (int64_t)0), (int64_t)INT32_MAX);
}

// Takes out what a mixed tile's columns do not see: their scores, the values of slots
// without a token, which may hold anything, NaN too, and infinities and NaN of any
// slot, since no weight of 0 takes those out.  Returns whether there were any: they go
// to the columns that see them later (add_nonfinite).
template <int DT, int CT, int DP, int C>
__device__ __forceinline__ bool mask_tile(const tree_args& a, const tree_span& r, int row, const int* t,
                                          const int* first, int tile, const bool* held, int lane,
                                          float (*p)[shape<DT, CT, DP>::kTokens],
                                          uint32_t (*v)[shape<DT, CT, DP>::kVWords]) {
  typedef shape<DT, CT, DP> S;
  // as if it were another number each time: nothing of this rare path is worth a register outside of it
  int lg = lane >> 4;
  asm volatile("" : "+v"(lg));
  uint32_t odd = 0;
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int u = 0; u < S::kSubs; ++u) {
      const int place = tile + 16 * u + 4 * lg;
      const uint32_t yes = column_sees(a, r, row, t[c], first[c], place);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        p[c][4 * u + j] = held[u] && place + j < r.len && (yes >> j & 1) ? p[c][4 * u + j] : -INFINITY;
    }
#pragma unroll
  for (int j = 0; j < S::kTokens; ++j) {
    const uint32_t keep = held[j / 4] && tile + 16 * (j / 4) + 4 * lg + j % 4 < r.len ? ~0u : 0u;
#pragma unroll
    for (int i = 0; i < S::kVWords; ++i) {
      v[j][i] &= keep;
      odd |= nonfinite_bits<DT, CT>(v[j][i]);
    }
  }
  if (!__any(odd)) return false;
#pragma unroll
  for (int j = 0; j < S::kTokens; ++j)
#pragma unroll
    for (int i = 0; i < S::kVWords; ++i) v[j][i] = finite_part<DT, CT>(v[j][i]);
  return true;
}

// The infinities and NaN among the values of a mixed tile, to the outputs of the columns
// that see them: whatever their weights, that is what comes out.
template <int DT, int CT, int DP, int C, bool FULL>
__device__ __forceinline__ void add_nonfinite(const tree_args& a, const tree_span& r, int row, const int* t,
                                              const int* first, int tile,
                                              const tile_place<shape<DT, CT, DP>::kSubs>& here, uint32_t value_slot,
                                              int lane, pl_f32x4 (*o)[shape<DT, CT, DP>::V]) {
  typedef shape<DT, CT, DP> S;
  const int lg = lane >> 4;
#pragma unroll 1
  for (int token = 0; token < S::kTile; ++token) {
    const int place = tile + token, u = token >> 4;
    if (place >= r.len || !(u ? here.held[S::kSubs - 1] : here.held[0])) continue;
    bool mine[C], any = false;
#pragma unroll
    for (int c = 0; c < C; ++c) mine[c] = column_sees(a, r, row, t[c], first[c], place) & 1, any = any || mine[c];
    const uintptr_t from = (u ? here.value[S::kSubs - 1] : here.value[0]) + (uint64_t)(token & 15) * value_slot;
#pragma unroll
    for (int n = 0; n < S::kPieces; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = S::value_at(4 * lg + e, n);
        uint32_t x[S::kVWords / S::kPieces] = {};
        if (any && (FULL || d < a.dim))
          __builtin_memcpy(x, reinterpret_cast<const void*>(from + d * S::kCsize), sizeof(x));
#pragma unroll
        for (int i = 0; i < S::kPiece; ++i) {
          const float y = value_element<DT, CT>(x, i), add = y - y == 0.f ? 0.f : y;
#pragma unroll
          for (int c = 0; c < C; ++c) o[c][n * S::kPiece + i][e] += mine[c] ? add : 0.f;
        }
        __builtin_amdgcn_sched_barrier(0);
      }
  }
}

// Raises the references of columns whose scores have gone far above them: the largest
// score takes the place.  They stay while no score is more than kSlack above them, so
// weights reach 2^kSlack, and the outputs are rescaled at a few tiles only.
template <int TOKENS, int V, int C, typename L>
__device__ __forceinline__ void rescale(const float (*p)[TOKENS], float scale2, float* m, L* l, pl_f32x4 (*o)[V]) {
  float top[C];
  bool beyond = false;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    top[c] = p[c][0];
#pragma unroll
    for (int j = 1; j < TOKENS; ++j) top[c] = fmaxf(top[c], p[c][j]);
    beyond = beyond || top[c] * scale2 > m[c] + kSlack;  // of this lane's tokens
  }
  if (!__any(beyond)) return;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    top[c] = fmaxf(column_max(top[c]) * scale2, m[c]);
    const float keep = exp2_fast(m[c] - (top[c] == -INFINITY ? 0.f : top[c]));
    l[c] *= keep;
#pragma unroll
    for (int i = 0; i < V; ++i) o[c][i] *= keep;
    m[c] = top[c];
  }
}

// Adds up a tile's values by the columns' weights, and the weights themselves, as the
// values of an element that is 1 everywhere: a product more on units that have little
// to do beside the vector unit (16-bit models).
template <int DT, int CT, int DP, int C>
__device__ __forceinline__ void add_values(const uint32_t (*v)[shape<DT, CT, DP>::kVWords],
                                           const pl_u32x4 (*part)[kWeightParts<DT>],
                                           pl_f32x4 (*o)[shape<DT, CT, DP>::V], pl_f32x4* l) {
  typedef shape<DT, CT, DP> S;
  constexpr uint32_t kOnes = DT == PL_BF16 ? 0x3f803f80u : 0x3c003c00u;
  const pl_u32x4 ones = {kOnes, kOnes, kOnes, kOnes};
#pragma unroll
  for (int k = 0; k < kWeightParts<DT>; ++k)
#pragma unroll
    for (int c = 0; c < C; ++c) l[c] = pl_mfma_chunk<DT>(ones, part[c][k], l[c]);
#pragma unroll
  for (int i = 0; i < S::V / 2; ++i) {
    uint32_t word[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (CT == PL_F8E4M3)
        word[j] = i % 2 ? widen<DT, true>(v[j][i / 2]) : widen<DT, false>(v[j][i / 2]);
      else
        word[j] = v[j][i];
    }
    pl_u32x4 x, y;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j] = __builtin_amdgcn_perm(word[2 * j + 1], word[2 * j], 0x05040100);
      y[j] = __builtin_amdgcn_perm(word[2 * j + 1], word[2 * j], 0x07060302);
    }
#pragma unroll
    for (int k = 0; k < kWeightParts<DT>; ++k)
#pragma unroll
      for (int c = 0; c < C; ++c) {
        o[c][2 * i] = pl_mfma_chunk<DT>(x, part[c][k], o[c][2 * i]);
        o[c][2 * i + 1] = pl_mfma_chunk<DT>(y, part[c][k], o[c][2 * i + 1]);
      }
    // in this order: pairing up all values first would take as many registers again
    __builtin_amdgcn_sched_barrier(0);
  }
}

// Four finished elements of a worker's column `in`.  A column without a token that counts
// went along where no tile was masked; no place seen gives 0; NaN, which no maximum
// shows, is in the sum and stays.
template <typename T, bool FULL>
__device__ __forceinline__ void put_output(const tree_args& a, int row, int col0, int in, int live, int hk, int d,
                                           pl_f32x4 x, float sum, float v_scale) {
  if (!FULL && d >= a.dim) return;
  x = in >= live || sum == 0.f ? pl_f32x4{0.f, 0.f, 0.f, 0.f} : x * (v_scale / sum);
  const column_place at = place_of(a, col0 + in, hk);
  store4((T*)a.out + (((int64_t)row * a.row_len + at.token) * a.heads + at.head) * a.dim + d, x);
}
// The same of a part; `sixteen` is the number of its first 16 columns.
template <int DP>
__device__ __forceinline__ void put_part(pl_buffer parts, int sixteen, int in, int d, pl_f32x4 x, float top,
                                         float sum) {
  typedef part_layout<DP> P;
  const uint32_t at = (uint32_t)(sixteen + in / kCols) * P::kBytes;
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(pl_u32x4, x), parts, at + P::at(in % kCols, d), 0,
                                         kAgentScope);
  if (d == 0)
    __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(pl_u32x2, pl_f32x2{top, sum}), parts,
                                          at + P::sums(in % kCols), 0, kAgentScope);
}

// Columns of a worker of the two kernels, by the padded head size.
constexpr int kWideWaves = 8;
constexpr int wide_columns(int dp) { return kWideWaves * kCols * (dp == 256 ? 1 : 2); }

}  // namespace

// The kernel for many columns (tree_wide.hip), 16-bit models.
int pl_tree_wide(int32_t dtype, int32_t cache_dtype, const tree_args& a, int64_t atoms_most, hipStream_t s);
