// Attention of drafted tokens over a paged key-value cache and over one another.
//
// Token t of row b looks at the row's tokens before the drafts (the last `window` of
// them counted from its own depth) and at those drafts that its mask names, itself
// among them:
//   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  s_j = scale * q . k_j,  m = max_j s_j,
// in one pass over keys and values, m, the sum and the unscaled output in fp32, as in
// paged_attention.hip, whose tiles these are.  The row's tokens times the query heads
// of a key head are the columns of the matrix products; a wave keeps C times 16 of
// them and reads each key and value once for all of them.
#include <type_traits>

#include "pl_attend.h"

namespace {

constexpr int kCus = 256;
constexpr int kWorkersMax = 2 * kCus;
constexpr int kXcdStep = kXcds;
constexpr int kColTilesMax = kWorkersMax / kXcds;

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
};

// Parts of 16 bits that a weight enters its product as.
template <int DT>
constexpr int kWeightParts = 2;

template <int DT, int CT, int DP, int C>
struct tree_state {
  typedef shape<DT, CT, DP> S;
  shared_u32x4* q;  // this lane's pieces, 64 apart
  pl_f32x4 o[C][S::V];
  float m[C], l[C];
  // this lane's column of each 16: its token (-1: none that counts) and the first place that it sees
  int t[C], first[C];
};

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
  r.first = live && a.window > 0 ? (int)max(first, (int64_t)0) : 0;
  r.base = r.first & ~31;
  r.atoms = max(1, (r.len - r.base + ATOM - 1) / ATOM);  // an empty row's output is an atom too
  return r;
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

// What an infinity or NaN among a tile's values does where some columns see its
// token and some do not: a product would put NaN into all of them.  So the
// products take the values without it, and it goes to the outputs of the
// columns that see it here, a token at a time.
template <int DT, int CT, int DP, int C>
__device__ __forceinline__ void add_nonfinite(tree_state<DT, CT, DP, C>& st, const tile_place<shape<DT, CT, DP>::kSubs>& at,
                                              uint32_t value_slot, int dim, const uint32_t (&alive)[C], int li, int lg) {
  typedef shape<DT, CT, DP> S;
#pragma unroll 1
  for (int token = 0; token < S::kTile; ++token) {
    const int u = token >> 4, from = ((token & 15) >> 2) * 16 + li, bit = u * 4 + (token & 3);
    uint32_t sees[C], any = 0;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      sees[c] = (uint32_t)__shfl((int)alive[c], from) >> bit & 1;
      any |= sees[c];
    }
    if (!__any(any)) continue;
    const uintptr_t p = (u ? at.value[S::kSubs - 1] : at.value[0]) + (uint64_t)(token & 15) * value_slot;
#pragma unroll
    for (int n = 0; n < S::kPieces; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = S::value_at(4 * lg + e, n);
        uint32_t x[S::kVWords / S::kPieces] = {};
        if (any && d < dim) __builtin_memcpy(x, __builtin_assume_aligned(reinterpret_cast<const void*>(p + d * S::kCsize), sizeof(x)), sizeof(x));
#pragma unroll
        for (int i = 0; i < S::kPiece; ++i) {
          const float y = value_element<DT, CT>(x, i), add = y - y == 0.f ? 0.f : y;
#pragma unroll
          for (int c = 0; c < C; ++c) st.o[c][n * S::kPiece + i][e] += sees[c] ? add : 0.f;
        }
        __builtin_amdgcn_sched_barrier(0);
      }
  }
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

template <int DT, int CT, int DP, int C, bool FULL, int WAVES_PER_SIMD>
__global__ __launch_bounds__(kThreads, WAVES_PER_SIMD) void pl_tree_attention_kernel(tree_args a) {
  typedef shape<DT, CT, DP> S;
  typedef typename pl_traits<DT>::T T;
  constexpr int kPad = 4, kParts = kWeightParts<DT>;
  __shared__ __attribute__((aligned(16))) float s_o[kWaves][kCols][DP + kPad];
  __shared__ __attribute__((aligned(16))) uint32_t s_q[C * S::kSteps * 64 * 4];
  __shared__ float s_m[kWaves][kCols], s_l[kWaves][kCols];
  __shared__ int s_last;
  const int tid = (int)threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int li = lane & 15, lg = lane >> 4;
  // Workers of one slice of tokens, one for each column tile, run side by side on one
  // XCD: the first to ask for a tile brings it into the L2 that the others read.
  const int round = (int)blockIdx.x / kXcdStep;
  const int ct = round % a.col_tiles;
  const int slice = (int)blockIdx.x % kXcdStep + kXcdStep * (round / a.col_tiles);

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
    const int n = span_of<S::kAtom>(a, pasts[k], counts[k]).atoms;
    atoms[k] = k * 64 + lane < a.rows ? n : 0;
    total += atoms[k], longest = max(longest, atoms[k]);
  }
  for (int b = kLooks * 64 + lane; b < a.rows; b += 64) {
    const int n = span_of<S::kAtom>(a, a.past[b], a.seq_lens ? a.seq_lens[b] : a.row_len).atoms;
    total += n, longest = max(longest, n);
  }
  total = __builtin_amdgcn_readlane(scan_sum(total), 63) * a.kv_heads;
  longest = __builtin_amdgcn_readlane(scan_max(longest), 63);
  const bool whole_pairs =
      choose_whole<S::kAtom / (kWaves * S::kTile)>(a.slices, total, a.rows * a.kv_heads, longest);
  const int per = (total + a.slices - 1) / a.slices;
  const int from = (int)min((int64_t)slice * per, (int64_t)total);
  const int to = min(total - per, from) + per;
  if (from >= total) return;
  // the row of its first atom: the first whose atoms up to and with it pass `from`
  int row = 0, row_start = 0, row_past = 0, row_new = 0, at = from;
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
      n = b < a.rows ? span_of<S::kAtom>(a, past, count).atoms : 0;
    }
    n *= a.kv_heads;
    const int upto = scan_sum(n) + row_start;
    const uint64_t passed = __ballot(upto > from);
    if (passed || b0 + 64 >= a.rows) {
      const int hit = passed ? __ffsll((long long)passed) - 1 : 63;
      row = b0 + hit;
      row_start = __builtin_amdgcn_readlane(upto - n, hit);
      row_past = __builtin_amdgcn_readlane(past, hit);
      row_new = __builtin_amdgcn_readlane(count, hit);
      break;
    }
    row_start = __builtin_amdgcn_readlane(upto, 63);
  }
  row = uniform(row);
  bool skip = whole_pairs;  // to the first pair that starts in the run
  while (at < to) {
    const tree_span r = span_of<S::kAtom>(a, row_past, row_new);
    int in_row = at - row_start;
    if (skip) {
      in_row = (in_row + r.atoms - 1) / r.atoms * r.atoms;
      at = row_start + in_row;
      skip = false;
      if (at >= to) return;
    }
    if (in_row >= r.atoms * a.kv_heads) {
      row_start += r.atoms * a.kv_heads;
      ++row;
      row_past = as_scalar(a.past)[row];
      row_new = a.seq_lens ? as_scalar(a.seq_lens)[row] : a.row_len;
      continue;
    }
    const int hk = in_row / r.atoms;
    const int pair_start = row_start + hk * r.atoms;
    const int first_atom = at - pair_start;
    const int last_atom = whole_pairs ? r.atoms : min(r.atoms, to - pair_start);
    // this worker's columns: tokens and heads of the launch's toks * group
    const int col0 = ct * C * kCols, cols_all = a.toks * a.group;

    tree_state<DT, CT, DP, C> st;
    st.q = reinterpret_cast<shared_u32x4*>(s_q) + lane;
    int all_from = 0;  // from this place on every column sees what lies before the drafts
    int last_t = -1;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      st.m[c] = -INFINITY, st.l[c] = 0.f;
#pragma unroll
      for (int i = 0; i < S::V; ++i) st.o[c][i] = pl_f32x4{0.f, 0.f, 0.f, 0.f};
      const int col = col0 + c * kCols + li;
      const int t = a.tok0 + col / a.group;
      st.t[c] = col < cols_all && t < r.n ? t : -1;
      st.first[c] = 0;
      if (a.window > 0 && st.t[c] >= 0) {
        const int depth = a.depths ? max(a.depths[row * a.depths_row + t], 0) : t;
        st.first[c] = (int)max((int64_t)r.past + depth - a.window + 1, (int64_t)0);
      }
      all_from = max(all_from, st.first[c]), last_t = max(last_t, st.t[c]);
    }
    if (a.window > 0) all_from = __builtin_amdgcn_readlane(scan_max(all_from), 63);
    // a line's last column sees the most; no column that counts, no token
    last_t = uniform(__builtin_amdgcn_readlane(scan_max(last_t + 1), 63));
    const float scale2 =
        a.scale * 1.44269504088896f * (CT == PL_F8E4M3 ? as_scalar(a.k_scale)[hk] : 1.f);

    // the queries, in the order of the products
    for (int i = tid; i < C * S::kSteps * 64; i += kThreads) {
      const int l = i & 63, n = (i >> 6) % S::kSteps, c = (i >> 6) / S::kSteps;
      const int g = l >> 4, col = col0 + c * kCols + (l & 15);
      const int d = CT == PL_F8E4M3 ? key_piece<CT>(n / 2, g, S::E) + (n % 2) * 8 : key_piece<CT>(n, g, S::E);
      pl_u32x4 x = {0, 0, 0, 0};
      if (col < cols_all && (FULL || d < a.dim)) {
        const int t = a.tok0 + col / a.group, h = hk * a.group + col % a.group;
        // rows of q have the alignment of their elements alone
        __builtin_memcpy(&x, (const T*)a.q + row * a.q_row + t * a.q_token + h * a.q_head + d, 16);
      }
      reinterpret_cast<shared_u32x4*>(s_q)[i] = x;
    }

    // the tiles of this wave: every fourth of the run's
    const int seen = a.visible ? r.len : (int)min((int64_t)r.len, (int64_t)r.past + last_t);
    const int end = last_t > 0 ? min(seen, r.base + last_atom * S::kAtom) : 0;
    constexpr int step = kWaves * S::kTile;
    walk w;
    w.key = reinterpret_cast<uintptr_t>(a.key.p) + (int64_t)hk * a.key.s_head * S::kCsize;
    w.value = reinterpret_cast<uintptr_t>(a.value.p) + (int64_t)hk * a.value.s_head * S::kCsize;
    w.pages = as_scalar(a.table.p + row * a.table.ld);
    w.key_page = a.key.s_page * S::kCsize, w.value_page = a.value.s_page * S::kCsize;
    w.key_slot = (uint32_t)a.key.s_slot * S::kCsize;
    w.value_slot = (uint32_t)a.value.s_slot * S::kCsize;
    w.end = end, w.shift = a.table.page_shift;
    w.num_pages = a.table.num_pages;
    // bytes from the first of 16 slots to the end of the last
    const uint32_t key_span = 15 * w.key_slot + (uint32_t)a.dim * S::kCsize;
    const uint32_t value_span = 15 * w.value_slot + (uint32_t)a.dim * S::kCsize;
    // lanes past the head's end ask for what no descriptor holds, and get 0
    constexpr uint32_t kNowhere = 0x80000000u;
    uint32_t key_off[S::kKeyLoads];
#pragma unroll
    for (int n = 0; n < S::kKeyLoads; ++n) {
      const int d = key_piece<CT>(n, lg, S::E);
      key_off[n] = FULL || d < a.dim ? li * w.key_slot + d * S::kCsize : kNowhere;
    }
    uint32_t value_off[S::kPieces];
#pragma unroll
    for (int n = 0; n < S::kPieces; ++n) {
      const int d = S::value_at(li, n);
      value_off[n] = FULL || d < a.dim ? 4 * lg * w.value_slot + d * S::kCsize : kNowhere;
    }
    // Loads as in paged_attention.hip: the next tile's keys behind this one's
    // scores, its values at its start, past the last tile loads of no bytes.
    auto load_keys = [&](pl_u32x4(&keys)[S::kSubs][S::kKeyLoads], const tile_place<S::kSubs>& at) {
#pragma unroll
      for (int u = 0; u < S::kSubs; ++u) {
        const pl_buffer b = make_buffer(at.key[u], at.held[u] ? key_span : 0);
#pragma unroll
        for (int n = 0; n < S::kKeyLoads; ++n) {
          uint32_t x[4];
          load_words<4, false>(b, key_off[n], 0, x);
          keys[u][n] = pl_u32x4{x[0], x[1], x[2], x[3]};
        }
      }
    };
    // One tile.  MIXED: not every column sees all of its tokens.
    pl_u32x4 keys[S::kSubs][S::kKeyLoads];
    tile_place<S::kSubs> place;
    int tile = r.base + first_atom * S::kAtom + wave * S::kTile;
    auto take_tile = [&](auto mixed) __attribute__((always_inline)) {
      constexpr bool MIXED = decltype(mixed)::value;
      uint32_t v[S::kTokens][S::kVWords];
#pragma unroll
      for (int u = 0; u < S::kSubs; ++u) {
        const pl_buffer b = make_buffer(place.value[u], place.held[u] ? value_span : 0);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int n = 0; n < S::kPieces; ++n)
            load_words<S::kVWords / S::kPieces, false>(b, value_off[n], j * w.value_slot,
                                                        v[4 * u + j] + n * (S::kVWords / S::kPieces));
      }
      const tile_place<S::kSubs> here = place;
      const int next = tile + step;
      place = place_tile<S::kSubs>(w, next);
      // scores, in units of log2 e
      float p[C][S::kTokens];
#pragma unroll
      for (int u = 0; u < S::kSubs; ++u) {
        pl_f32x4 s[C];
#pragma unroll
        for (int c = 0; c < C; ++c) s[c] = pl_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < S::kKeyLoads; ++n) {
          const pl_u32x4 k = keys[u][n];
          if constexpr (CT == PL_F8E4M3) {
            const pl_u32x4 x = {widen<DT, false>(k.x), widen<DT, true>(k.x), widen<DT, false>(k.y),
                                widen<DT, true>(k.y)};
            const pl_u32x4 y = {widen<DT, false>(k.z), widen<DT, true>(k.z), widen<DT, false>(k.w),
                                widen<DT, true>(k.w)};
#pragma unroll
            for (int c = 0; c < C; ++c) s[c] = pl_mfma_chunk<DT>(x, st.q[(c * S::kSteps + 2 * n) * 64], s[c]);
#pragma unroll
            for (int c = 0; c < C; ++c) s[c] = pl_mfma_chunk<DT>(y, st.q[(c * S::kSteps + 2 * n + 1) * 64], s[c]);
          } else if (DT != PL_F32 || FULL || n * 4 * S::E < a.dim) {
#pragma unroll
            for (int c = 0; c < C; ++c) s[c] = pl_mfma_chunk<DT>(k, st.q[(c * S::kSteps + n) * 64], s[c]);
          }
        }
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int j = 0; j < 4; ++j) p[c][4 * u + j] = s[c][j] * scale2;
      }
      load_keys(keys, place);
      uint32_t alive[C];
      bool nonfinite = false;
      if constexpr (MIXED) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
          alive[c] = 0;
          const int32_t* bits = a.visible + row * a.visible_row + max(st.t[c], 0) * a.visible_token;
#pragma unroll
          for (int j = 0; j < S::kTokens; ++j) {
            const int token = tile + 16 * (j / 4) + 4 * lg + j % 4, draft = token - r.past;
            bool sees = here.held[j / 4] && token < r.len && st.t[c] >= 0;
            if (draft < 0)
              sees = sees && token >= st.first[c];
            else if (!a.visible)
              sees = sees && token >= st.first[c] && draft <= st.t[c];
            else if (sees)
              sees = bits[draft >> 5] >> (draft & 31) & 1;
            p[c][j] = sees ? p[c][j] : -INFINITY;
            alive[c] |= (uint32_t)sees << j;
          }
        }
        // slots without a token may hold anything, NaN too: no weight of 0 takes that out
#pragma unroll
        for (int j = 0; j < S::kTokens; ++j) {
          const bool holds = here.held[j / 4] && tile + 16 * (j / 4) + 4 * lg + j % 4 < r.len;
#pragma unroll
          for (int i = 0; i < S::kVWords; ++i) {
            v[j][i] = holds ? v[j][i] : 0u;
            nonfinite = nonfinite || finite_part<DT, CT>(v[j][i]) != v[j][i];
          }
        }
        nonfinite = __any(nonfinite);
        if (nonfinite) {
#pragma unroll
          for (int j = 0; j < S::kTokens; ++j)
#pragma unroll
            for (int i = 0; i < S::kVWords; ++i) v[j][i] = finite_part<DT, CT>(v[j][i]);
        }
      }
      // the running maximum and sum, and the weights
      pl_u32x4 part[C][kParts];
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float top = p[c][0];
#pragma unroll
        for (int j = 1; j < S::kTokens; ++j) top = fmaxf(top, p[c][j]);
        top = fmaxf(st.m[c], column_max(top));
        // nothing alive yet: any finite reference gives weights of 0
        const float ref = top == -INFINITY ? 0.f : top;
        if (__any(top > st.m[c])) {
          const float keep = exp2_fast(st.m[c] - ref);
          st.l[c] *= keep;
#pragma unroll
          for (int i = 0; i < S::V; ++i) st.o[c][i] *= keep;
          st.m[c] = top;
        }
#pragma unroll
        for (int j = 0; j < S::kTokens; ++j) {
          p[c][j] = exp2_fast(S::kLift ? p[c][j] - ref + S::kLift : p[c][j] - ref);
          st.l[c] += p[c][j];
        }
        if constexpr (DT != PL_F32) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float x = p[c][2 * j], y = p[c][2 * j + 1];
#pragma unroll
            for (int k = 0; k < kParts; ++k) {
              const uint32_t z = k + 1 < kParts ? pack2_down<DT>(x, y) : pack2<DT>(x, y);
              if (k + 1 < kParts) x -= unpack<DT>(z, 0), y -= unpack<DT>(z, 1);
              // no part negative, or 0 beside the others: an infinite value stays one
              part[c][k][j] = k ? at_least_smallest<DT>(z, part[c][0][j]) : z;
            }
          }
        }
      }
      if constexpr (MIXED)
        if (nonfinite) add_nonfinite<DT, CT, DP, C>(st, here, w.value_slot, a.dim, alive, li, lg);
      if constexpr (DT == PL_F32) {
#pragma unroll
        for (int i = 0; i < S::V; ++i) {
#pragma unroll
          for (int c = 0; c < C; ++c) {
            pl_f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < S::kTokens; ++j)
              sum = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v[j][i]), p[c][j], sum, 0, 0, 0);
            st.o[c][i] += sum;
          }
          if (i % 2) __builtin_amdgcn_sched_barrier(0);
        }
      } else {
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
          for (int k = 0; k < kParts; ++k)
#pragma unroll
            for (int c = 0; c < C; ++c) {
              st.o[c][2 * i] = pl_mfma_chunk<DT>(x, part[c][k], st.o[c][2 * i]);
              st.o[c][2 * i + 1] = pl_mfma_chunk<DT>(y, part[c][k], st.o[c][2 * i + 1]);
            }
          // in this order: pairing up all values first would take as many registers again
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      tile = next;
    };
    __syncthreads();
    if (tile < end) {
      place = place_tile<S::kSubs>(w, tile);
      load_keys(keys, place);
      do {
        bool whole = tile >= all_from && tile + S::kTile <= min(r.past, r.len);
#pragma unroll
        for (int u = 0; u < S::kSubs; ++u) whole = whole && place.held[u];
        if (__builtin_expect(whole, 1))
          take_tile(std::false_type{});
        else
          take_tile(std::true_type{});
      } while (tile < end);
    }

    // join the waves, 16 columns at a time
    const float v_scale = CT == PL_F8E4M3 ? as_scalar(a.v_scale)[hk] : 1.f;
    const bool complete = first_atom == 0 && last_atom == r.atoms;
    typedef part_layout<DP> P;
    const int slot = 2 * (slice * a.col_tiles + ct) + (at == from ? 0 : 1);
    const pl_buffer parts = P::all(a.parts, 2u * kWorkersMax * C);
    auto finish = [&](int c, int i, int d, pl_f32x4 x) {
      const int col = col0 + c * kCols + i;
      if (col >= cols_all || !(FULL || d < a.dim)) return;
      const int t = a.tok0 + col / a.group, h = hk * a.group + col % a.group;
      // a column without a token that counts went along where no tile was masked
      if (t >= r.n) x = pl_f32x4{0.f, 0.f, 0.f, 0.f};
      store4((T*)a.out + (((int64_t)row * a.row_len + t) * a.heads + h) * a.dim + d, x);
    };
#pragma unroll
    for (int c = 0; c < C; ++c) {
      st.l[c] = column_sum(st.l[c]);
      if (c > 0) __syncthreads();
      if (lg == 0) s_m[wave][li] = st.m[c], s_l[wave][li] = st.l[c];
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int i = 0; i < S::V; i += 4)
          *reinterpret_cast<pl_f32x4*>(&s_o[wave][li][S::value_at(4 * lg + e, i / S::kPiece) + i % S::kPiece]) =
              pl_f32x4{st.o[c][i][e], st.o[c][i + 1][e], st.o[c][i + 2][e], st.o[c][i + 3][e]};
      __syncthreads();
      const uint32_t part = (uint32_t)(slot * C + c) * P::kBytes;
      for (int i = tid; i < kCols * (DP / 4); i += kThreads) {
        const int col = i / (DP / 4), d = i % (DP / 4) * 4;
        float m = -INFINITY, l = 0.f;
        pl_f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < kWaves; ++k) m = fmaxf(m, s_m[k][col]);
        const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int k = 0; k < kWaves; ++k) {
          const float f = exp2_fast(s_m[k][col] - ref);
          l += f * s_l[k][col];
          o += f * *reinterpret_cast<const pl_f32x4*>(&s_o[k][col][d]);
        }
        if (complete) {
          // no token gives 0; NaN, which no maximum shows, is in l and stays
          finish(c, col, d, l == 0.f ? pl_f32x4{0.f, 0.f, 0.f, 0.f} : o * (v_scale / l));
        } else {
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(pl_u32x4, o), parts, part + P::at(col, d), 0,
                                                 kAgentScope);
          if (d == 0)
            __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(pl_u32x2, pl_f32x2{m, l}), parts,
                                                  part + P::sums(col), 0, kAgentScope);
        }
      }
    }
    if (!complete) {
      // Parts are acknowledged from where every XCD sees them before the arrival
      // is counted, and the last to arrive asks for them there after that.
      const int w0 = pair_start / per, w1 = (pair_start + r.atoms - 1) / per;
      __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
      __syncthreads();
      if (tid == 0) {
        int32_t* counter = a.counters + (w0 * a.col_tiles + ct) * kCounterStride;
        const int old = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        s_last = old == w1 - w0;
        if (s_last) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
      __syncthreads();
      if (s_last) {
        // the first part is its workgroup's second when that workgroup began earlier
        const int slot1 = 2 * (w0 * a.col_tiles + ct), slot0 = slot1 + (w0 * per == pair_start ? 0 : 1);
        for (int c = 0; c < C; ++c)
          join_parts<DP>(parts, slot0 * C + c, slot1 * C + c, 2 * a.col_tiles * C, w1 - w0 + 1, kCols, &s_o[0][0][0],
                         [&](int i, int d, pl_f32x4 x) { finish(c, i, d, x * v_scale); });
      }
    }
    __syncthreads();  // the shared arrays are free again
    at = pair_start + last_atom;
  }
}

// Columns of a worker, in sixteens, and the waves of a SIMD that it is built for.
template <int DT, int CT, int DP, int C, int WAVES_PER_SIMD>
void launch_columns(tree_args a, int64_t atoms_most, hipStream_t s) {
  const int columns = a.toks * a.group;
  a.col_tiles = (columns + C * kCols - 1) / (C * kCols);
  const int64_t most = kCus * WAVES_PER_SIMD / (kXcdStep * a.col_tiles), need = (atoms_most + kXcdStep - 1) / kXcdStep;
  a.slices = kXcdStep * (int)(need < most ? need : most > 0 ? most : 1);
  const dim3 grid((unsigned)(a.slices * a.col_tiles));
  if (a.dim == DP)
    pl_tree_attention_kernel<DT, CT, DP, C, true, WAVES_PER_SIMD><<<grid, kThreads, 0, s>>>(a);
  else
    pl_tree_attention_kernel<DT, CT, DP, C, false, WAVES_PER_SIMD><<<grid, kThreads, 0, s>>>(a);
}

// Columns of the widest worker.
template <int DT>
constexpr int columns_most(int dim) {
  return DT == PL_F32 || dim > 128 ? 2 * kCols : 4 * kCols;
}

template <int DT, int CT, int DP>
void launch_dim(const tree_args& a, int64_t atoms_most, hipStream_t s) {
  const int columns = a.toks * a.group;
  if (columns <= kCols)
    launch_columns<DT, CT, DP, 1, DP == 256 ? 1 : 2>(a, atoms_most, s);
  else if (columns <= 2 * kCols || DT == PL_F32 || DP == 256)
    launch_columns<DT, CT, DP, 2, DT == PL_F32 || DP == 256 ? 1 : 2>(a, atoms_most, s);
  else if constexpr (DT != PL_F32 && DP <= 128)
    launch_columns<DT, CT, DP, 4, 1>(a, atoms_most, s);
}

template <int DT, int CT>
int launch(tree_args a, int64_t atoms_most, hipStream_t s) {
  // tokens of a launch: as many columns as there are workers for
  const int toks = kColTilesMax * columns_most<DT>(a.dim) / a.group;
  for (a.tok0 = 0; a.tok0 < a.row_len; a.tok0 += toks) {
    a.toks = a.row_len - a.tok0 < toks ? a.row_len - a.tok0 : toks;
    if (a.dim <= 64)
      launch_dim<DT, CT, 64>(a, atoms_most, s);
    else if (a.dim <= 128)
      launch_dim<DT, CT, 128>(a, atoms_most, s);
    else
      launch_dim<DT, CT, 256>(a, atoms_most, s);
    const int rc = pl_launch_status("pl_tree_attention");
    if (rc) return rc;
  }
  return PL_OK;
}

}  // namespace

static_assert(PL_ATTENTION_COUNTER_INTS == kWorkersMax * kCounterStride, "one counter per workgroup");

extern "C" int64_t pl_tree_attention_workspace_bytes(int32_t dim) {
  const int dp = dim <= 64 ? 64 : dim <= 128 ? 128 : 256, c = dp == 256 ? 2 : 4;
  return dim < 1 || dim > kHeadDimMax ? 0 : 2ll * kWorkersMax * c * part_floats(dp) * (int64_t)sizeof(float);
}

extern "C" int pl_tree_attention(int32_t dtype, int32_t cache_dtype, const void* q, const int64_t* q_strides,
                                 const void* key_cache, const int64_t* key_strides, const void* value_cache,
                                 const int64_t* value_strides, int32_t num_pages, int32_t page_size,
                                 const int32_t* page_table, int64_t table_ld, int32_t max_pages,
                                 const int32_t* past_lens, const int32_t* seq_lens, const int32_t* visible,
                                 int64_t visible_row, int64_t visible_token, int32_t words, const int32_t* depths,
                                 int64_t depths_row, int32_t rows, int32_t row_len, int32_t heads, int32_t kv_heads,
                                 int32_t dim, float scale, int32_t window, const float* k_scale, const float* v_scale,
                                 void* out, void* workspace, int64_t workspace_bytes, int32_t* counters,
                                 int64_t counter_ints, void* stream) {
  const char* what = "pl_tree_attention";
  const int rc = pl_check_paged(what, dtype, cache_dtype, key_cache, key_strides, value_cache, value_strides,
                                num_pages, page_size, page_table, table_ld, max_pages, rows, heads, kv_heads, dim,
                                k_scale, v_scale);
  if (rc) return rc;
  if (row_len < 0 || window < 0 || (visible && (int64_t)words * 32 < row_len)) {
    pl_set_error("%s: bad sizes (row_len %d, window %d, %d words to a mask)", what, row_len, window, words);
    return PL_ERR_ARG;
  }
  if (window > 0 && visible && (!depths || window < row_len)) {
    pl_set_error("%s: a window over a tree needs depths and at least the drafts' number of tokens (got %d, %d)", what,
                 window, row_len);
    return PL_ERR_ARG;
  }
  const int64_t tokens = (int64_t)rows * row_len;
  if (tokens == 0) return PL_OK;
  if (heads / kv_heads > kColTilesMax * 2 * kCols) {
    pl_set_error("%s: at most %d query heads to a key head (got %d)", what, kColTilesMax * 2 * kCols, heads / kv_heads);
    return PL_ERR_LIMIT;
  }
  // lanes address the 16 slots of a tile with 32-bit byte offsets
  const int64_t slot_most = INT32_MAX / 16 / pl_cache_elem_size(cache_dtype);
  if (key_strides[2] < 0 || key_strides[2] > slot_most || value_strides[2] < 0 || value_strides[2] > slot_most) {
    pl_set_error("%s: slot strides of %lld and %lld elements", what, (long long)key_strides[2],
                 (long long)value_strides[2]);
    return PL_ERR_LIMIT;
  }
  if (!q || !q_strides || !past_lens || !out) {
    pl_set_error("%s: null pointer", what);
    return PL_ERR_ARG;
  }
  const int64_t es = pl_elem_size(dtype);
  const int64_t reach = (rows - 1) * q_strides[0] + (row_len - 1) * q_strides[1] + (heads - 1) * q_strides[2] + dim;
  if (pl_ranges_meet(out, tokens * heads * dim * es, q, reach * es)) {
    pl_set_error("%s: out overlaps q", what);
    return PL_ERR_ARG;
  }
  if (!workspace || workspace_bytes < pl_tree_attention_workspace_bytes(dim) || !counters ||
      counter_ints < PL_ATTENTION_COUNTER_INTS) {
    pl_set_error("%s: workspace of %lld bytes and %lld counters, %lld and %d needed", what, (long long)workspace_bytes,
                 (long long)counter_ints, (long long)pl_tree_attention_workspace_bytes(dim), PL_ATTENTION_COUNTER_INTS);
    return PL_ERR_ARG;
  }
  tree_args a;
  a.q = q, a.q_row = q_strides[0], a.q_token = q_strides[1], a.q_head = q_strides[2];
  a.key = {const_cast<void*>(key_cache), key_strides[0], key_strides[1], key_strides[2]};
  a.value = {const_cast<void*>(value_cache), value_strides[0], value_strides[1], value_strides[2]};
  a.table = {page_table, table_ld, max_pages, num_pages, pl_log2_exact(page_size)};
  a.past = past_lens, a.seq_lens = seq_lens, a.visible = visible, a.visible_row = visible_row;
  a.visible_token = visible_token, a.depths = visible ? depths : nullptr, a.depths_row = depths_row;
  a.k_scale = k_scale, a.v_scale = v_scale, a.out = out, a.scale = scale, a.rows = rows, a.row_len = row_len;
  a.heads = heads, a.kv_heads = kv_heads, a.dim = dim, a.window = window, a.group = heads / kv_heads;
  a.parts = static_cast<float*>(workspace), a.counters = counters;
  // atoms at most: every row as long as its pages or its window allow
  int64_t longest = (int64_t)max_pages * page_size;
  if (window > 0 && longest > (int64_t)window + row_len + 31) longest = (int64_t)window + row_len + 31;
  const int64_t atom = 32 * kWaves, per_pair = longest > atom ? (longest + atom - 1) / atom : 1;
  const int64_t pairs = (int64_t)rows * kv_heads;
  // token and atom numbers are 32-bit, a tile past a row's end and a run past the last one included
  if ((int64_t)max_pages * page_size > INT32_MAX - 2 * atom || pairs > (INT32_MAX - kWorkersMax) / per_pair) {
    pl_set_error("%s: %lld rows and key heads of up to %lld tokens are too many", what, (long long)pairs,
                 (long long)longest);
    return PL_ERR_LIMIT;
  }
  const int64_t atoms_most = pairs * per_pair;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (cache_dtype == PL_F8E4M3)
    return dtype == PL_BF16 ? launch<PL_BF16, PL_F8E4M3>(a, atoms_most, s) : launch<PL_F16, PL_F8E4M3>(a, atoms_most, s);
  if (dtype == PL_F32) return launch<PL_F32, PL_F32>(a, atoms_most, s);
  return dtype == PL_BF16 ? launch<PL_BF16, PL_BF16>(a, atoms_most, s) : launch<PL_F16, PL_F16>(a, atoms_most, s);
}
