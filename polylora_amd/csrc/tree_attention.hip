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
//
// Few columns are bound by memory, more by the chain from a tile's scores to its weights to
// its products.  Measured, bf16, 32 query heads over 8 of 128: 8 tokens of 64 rows over up
// to 4096 (C = 2) 155 us, 3.6 TB/s; 4 tokens (C = 1) 113 us, 4.9 TB/s; 6 tokens of one row over
// 700 14.2 us, a chain of reads and the waves' join; 16 tokens over 131072 in 8 bits 103 us.
#include "pl_tree.h"

namespace {

// Workgroups on a CU, by the registers and the LDS that they take: a wave of 16-bit models
// holds 32 columns' outputs, queries and two tiles on their way in 256 registers; fp32's
// queries and the outputs of heads above 128 elements need more.
template <int DT, int DP, int C>
constexpr int waves_per_simd() {
  return DP == 256 || (DT == PL_F32 && DP == 128 && C == 2) ? 1 : 2;
}

template <int DT, int CT, int DP, int C, bool FULL, bool STREAM>
__global__ __launch_bounds__(kThreads, (waves_per_simd<DT, DP, C>())) void pl_tree_attention_kernel(tree_args a) {
  typedef shape<DT, CT, DP> S;
  typedef typename pl_traits<DT>::T T;
  constexpr int kPitch = DP + 4, kParts = kWeightParts<DT>, kColumns = C * kCols;
  constexpr float kLift = DT == PL_F16 ? 15.f - kSlack : 0.f;
  constexpr bool kQueryLds = DT == PL_F32;  // its pieces are twice as many
  __shared__ __attribute__((aligned(16))) float s_o[kWaves * kColumns * kPitch];
  __shared__ __attribute__((aligned(16))) uint32_t s_q[kQueryLds ? C * S::kSteps * 64 * 4 : 4];
  __shared__ float s_m[kWaves][kColumns], s_l[kWaves][kColumns];
  __shared__ int s_last;
  const int tid = (int)threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int li = lane & 15, lg = lane >> 4;
  const tree_worker me = worker_of(a);
  const int ct = me.ct, slice = me.slice;
  const tree_run run = find_run<S::kAtom, S::kAtom / (kWaves * S::kTile)>(
      a, slice, lane, DT != PL_F32 && DP <= 128 && C == 1 && a.dim * S::kCsize >= 128 && a.col_tiles == 1);
  const int from = run.from, to = run.to, per = run.per;
  const bool whole_pairs = run.whole_pairs;
  if (from >= run.total) return;
  int row = run.row, row_start = run.row_start, row_past = run.row_past, row_new = run.row_new, at = from;
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
    // this worker's columns: tokens and heads of the launch's toks * group, and those of tokens that count
    const int col0 = ct * kColumns, cols = min(kColumns, a.toks * a.group - col0);
    const int live = max(0, min(cols, (min(r.n, a.tok0 + a.toks) - a.tok0) * a.group - col0));

    // The scale's sign goes into the queries: the largest score is the largest product.
    // (0 as the smallest factor, so that masked scores of -infinity stay that.)
    const float signed_scale = a.scale * 1.44269504088896f * (CT == PL_F8E4M3 ? as_scalar(a.k_scale)[hk] : 1.f);
    const float scale2 = fmaxf(fabsf(signed_scale), 1.17549435e-38f);
    const uint32_t flip = signed_scale < 0.f ? DT == PL_F32 ? 0x80000000u : 0x80008000u : 0u;
    pl_u32x4 q_own[kQueryLds ? 1 : C][kQueryLds ? 1 : S::kSteps];
    shared_u32x4* q_lds = reinterpret_cast<shared_u32x4*>(s_q) + lane;
    pl_f32x4 o[C][S::V];
    float m[C];
    typename std::conditional<DT == PL_F32, float, pl_f32x4>::type l[C];  // fp32: of this lane's tokens
    // this lane's column of each 16: its token (-1: none that counts) and the first place that it sees
    int t[C], first[C], all_from = 0;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      m[c] = -INFINITY, l[c] = {};
#pragma unroll
      for (int i = 0; i < S::V; ++i) o[c][i] = pl_f32x4{0.f, 0.f, 0.f, 0.f};
      const int in = c * kCols + li;
      const column_place at = place_of(a, col0 + in, hk);
      t[c] = in < live ? at.token : -1;
      first[c] = first_seen(a, r, row, t[c]);
      all_from = max(all_from, first[c]);
      const T* q = (const T*)a.q + row * a.q_row + at.token * a.q_token + at.head * a.q_head;
      // (all waves write the same where they share them)
#pragma unroll
      for (int n = 0; n < S::kSteps; ++n) {
        const int d = CT == PL_F8E4M3 ? key_piece<CT>(n / 2, lg, S::E) + (n % 2) * 8 : key_piece<CT>(n, lg, S::E);
        pl_u32x4 x = {0, 0, 0, 0};
        // rows of q have the alignment of their elements alone
        if (in < live && (FULL || d < a.dim)) __builtin_memcpy(&x, q + d, 16);
        if constexpr (kQueryLds)
          q_lds[(c * S::kSteps + n) * 64] = x ^ flip;
        else
          q_own[c][n] = x ^ flip;
      }
    }
    auto query = [&](int c, int n) __attribute__((always_inline)) {
      if constexpr (kQueryLds)
        return q_lds[(c * S::kSteps + n) * 64];
      else
        return q_own[c][n];
    };
    if (a.window > 0) all_from = __builtin_amdgcn_readlane(scan_max(all_from), 63);

    // the tiles of this wave: every fourth of the run's; a line's last column sees the most
    const int last_t = place_of(a, max(0, col0 + live - 1), hk).token;
    const int seen = a.visible ? r.len : (int)min((int64_t)r.len, (int64_t)r.past + uniform(last_t) + 1);
    const int end = live > 0 ? min(seen, r.base + last_atom * S::kAtom) : 0;
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
    pl_u32x4 keys[S::kSubs][S::kKeyLoads];
    bool nonfinite = false;  // values of a mixed tile were infinities or NaN
    const int first_tile = r.base + first_atom * S::kAtom + wave * S::kTile;
    // not every column sees all of a mixed tile's tokens
    auto mixed = [&](int tile, const tile_place<S::kSubs>& here) __attribute__((always_inline)) {
      bool no = tile < all_from || tile + S::kTile > min(r.past, r.len);
#pragma unroll
      for (int u = 0; u < S::kSubs; ++u) no = no || !here.held[u];
      return no;
    };
    auto load_keys = [&](const tile_place<S::kSubs>& from) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < S::kSubs; ++u) {
        const pl_buffer b = make_buffer(from.key[u], from.held[u] ? key_span : 0);
#pragma unroll
        for (int n = 0; n < S::kKeyLoads; ++n) {
          uint32_t x[4];
          load_words<4, STREAM>(b, key_off[n], 0, x);
          keys[u][n] = pl_u32x4{x[0], x[1], x[2], x[3]};
        }
      }
    };
    if (first_tile < end) {
      tile_place<S::kSubs> place = place_tile<S::kSubs>(w, first_tile);
      load_keys(place);
      int tile = first_tile;
      do {
        uint32_t v[S::kTokens][S::kVWords];
#pragma unroll
        for (int u = 0; u < S::kSubs; ++u) {
          const pl_buffer b = make_buffer(place.value[u], place.held[u] ? value_span : 0);
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int n = 0; n < S::kPieces; ++n)
              load_words<S::kVWords / S::kPieces, STREAM>(b, value_off[n], j * w.value_slot,
                                                          v[4 * u + j] + n * (S::kVWords / S::kPieces));
        }
        const tile_place<S::kSubs> here = place;
        const int next = tile + step;
        place = place_tile<S::kSubs>(w, next);
        float p[C][S::kTokens];  // scores, without the scale
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
              for (int c = 0; c < C; ++c) s[c] = pl_mfma_chunk<DT>(x, query(c, 2 * n), s[c]);
#pragma unroll
              for (int c = 0; c < C; ++c) s[c] = pl_mfma_chunk<DT>(y, query(c, 2 * n + 1), s[c]);
            } else if (DT != PL_F32 || FULL || n * 4 * S::E < a.dim) {
#pragma unroll
              for (int c = 0; c < C; ++c) s[c] = pl_mfma_chunk<DT>(k, query(c, n), s[c]);
            }
          }
#pragma unroll
          for (int c = 0; c < C; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) p[c][4 * u + j] = s[c][j];
        }
        load_keys(place);
        if (mixed(tile, here)) nonfinite |= mask_tile<DT, CT, DP, C>(a, r, row, t, first, tile, here.held, lane, p, v);
        rescale<S::kTokens, S::V, C>(p, scale2, m, l, o);
        pl_u32x4 part[C][kParts];
#pragma unroll
        for (int c = 0; c < C; ++c) {
          // nothing alive yet: any finite reference gives weights of 0
          const float ref = (m[c] == -INFINITY ? 0.f : m[c]) - kLift;
#pragma unroll
          for (int j = 0; j < S::kTokens; ++j) {
            p[c][j] = exp2_fast(fmaf(p[c][j], scale2, -ref));
            if constexpr (DT == PL_F32) l[c] += p[c][j];
          }
          if constexpr (DT != PL_F32) weight_parts<DT>(p[c], part[c]);
        }
        if constexpr (DT == PL_F32) {
#pragma unroll
          for (int i = 0; i < S::V; ++i) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
              pl_f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int j = 0; j < S::kTokens; ++j)
                sum = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v[j][i]), p[c][j], sum, 0, 0, 0);
              o[c][i] += sum;
            }
            if (i % 2) __builtin_amdgcn_sched_barrier(0);
          }
        } else {
          add_values<DT, CT, DP, C>(v, part, o, l);
        }
        tile = next;
      } while (tile < end);
      if (__builtin_expect(nonfinite, 0))
        for (tile = first_tile; tile < end; tile += step) {
          const tile_place<S::kSubs> here = place_tile<S::kSubs>(w, tile);
          if (mixed(tile, here))
            add_nonfinite<DT, CT, DP, C, FULL>(a, r, row, t, first, tile, here, w.value_slot, lane, o);
        }
    }

    // join the waves
    const float v_scale = CT == PL_F8E4M3 ? as_scalar(a.v_scale)[hk] : 1.f;
    const bool complete = first_atom == 0 && last_atom == r.atoms;
    typedef part_layout<DP> P;
    const int slot = 2 * (slice * a.col_tiles + ct) + (at == from ? 0 : 1);
    const pl_buffer parts = P::all(a.parts, 2u * kWorkersMax * C);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float sum;
      if constexpr (DT == PL_F32)
        sum = column_sum(l[c]);
      else
        sum = l[c].x;
      if (lg == 0) s_m[wave][c * kCols + li] = m[c], s_l[wave][c * kCols + li] = sum;
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int i = 0; i < S::V; i += 4)
          *reinterpret_cast<pl_f32x4*>(s_o + (wave * kColumns + c * kCols + li) * kPitch +
                                       S::value_at(4 * lg + e, i / S::kPiece) + i % S::kPiece) =
              pl_f32x4{o[c][i][e], o[c][i + 1][e], o[c][i + 2][e], o[c][i + 3][e]};
    }
    __syncthreads();
    // columns past the last are no column's, and of one without a token that counts 0 comes out
    for (int i = tid; i < cols * (DP / 4); i += kThreads) {
      const int in = i / (DP / 4), d = i % (DP / 4) * 4;
      float top = -INFINITY, sum = 0.f;
      pl_f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < kWaves; ++k) top = fmaxf(top, s_m[k][in]);
      const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int k = 0; k < kWaves; ++k) {
        const float f = exp2_fast(s_m[k][in] - ref);
        sum += f * s_l[k][in];
        x += f * *reinterpret_cast<const pl_f32x4*>(s_o + (k * kColumns + in) * kPitch + d);
      }
      if (complete)
        put_output<T, FULL>(a, row, col0, in, live, hk, d, x, sum, v_scale);
      else
        put_part<DP>(parts, slot * C, in, d, x, top, sum);
    }
    if (!complete) {
      const int w0 = pair_start / per, w1 = (pair_start + r.atoms - 1) / per;
      if (arrive_last(a.counters + (w0 * a.col_tiles + ct) * kCounterStride, w1 - w0, &s_last)) {
        // the first part is its workgroup's second when that workgroup began earlier
        const int slot1 = 2 * (w0 * a.col_tiles + ct), slot0 = slot1 + (w0 * per == pair_start ? 0 : 1);
        for (int c = 0; c < C; ++c)
          join_parts<DP>(parts, slot0 * C + c, slot1 * C + c, 2 * a.col_tiles * C, w1 - w0 + 1, kCols, s_o,
                         [&](int i, int d, pl_f32x4 x) {
                           if (c * kCols + i < cols)
                             put_output<T, FULL>(a, row, col0, c * kCols + i, live, hk, d, x, 1.f, v_scale);
                         });
      }
    }
    __syncthreads();  // the shared arrays are free again
    at = pair_start + last_atom;
  }
}

constexpr int kColTilesMax = kWorkersMax / kXcds;

// Columns of a worker, in sixteens.
template <int DT, int CT, int DP, int C>
void launch_columns(tree_args a, int64_t atoms_most, hipStream_t s) {
  const int columns = a.toks * a.group;
  a.col_tiles = (columns + C * kCols - 1) / (C * kCols);
  a.once = a.once && a.col_tiles == 1;
  a.slices = slices_of(atoms_most, kCus * waves_per_simd<DT, DP, C>(), a.col_tiles);
  const dim3 grid((unsigned)(a.slices * a.col_tiles));
  if (a.dim != DP)
    pl_tree_attention_kernel<DT, CT, DP, C, false, false><<<grid, kThreads, 0, s>>>(a);
  else if (a.once)
    pl_tree_attention_kernel<DT, CT, DP, C, true, true><<<grid, kThreads, 0, s>>>(a);
  else
    pl_tree_attention_kernel<DT, CT, DP, C, true, false><<<grid, kThreads, 0, s>>>(a);
}

// Columns above which 16-bit models take the other kernel, which reads keys and values
// once for all of them where this one reads them again for each 32 (16 of heads above
// 128 elements), out of the XCD's cache mostly.  Measured in us, this one and the other, 64 rows
// over 4096 tokens, 8 key heads of 128: 36 columns 183 and 209, 64 185 and 215, 96 223 and
// 263, 128 262 and 273 (252 with weights in two parts); one row over 700: 64 columns 15.9 and 22, 128 16.4
// and 24; one over 131072 in 8 bits: 64 columns 110 and 129, 96 143 and 182, 128 175 and 184.  Heads of 256
// elements: 32 columns 299 and 292, one row 15.5 and 23, 8 bits 131 and 163; 64 columns 494 and 320.
constexpr int narrow_columns(int dp) { return dp == 256 ? 2 * kCols : 6 * kCols; }

template <int DT, int CT, int DP>
int launch_dim(int32_t dtype, int32_t cache_dtype, const tree_args& a, int64_t atoms_most, hipStream_t s) {
  const int columns = a.toks * a.group;
  if (DT != PL_F32 && columns > narrow_columns(DP)) return pl_tree_wide(dtype, cache_dtype, a, atoms_most, s);
  if constexpr (DP == 256)
    launch_columns<DT, CT, DP, 1>(a, atoms_most, s);
  else if (columns <= kCols)
    launch_columns<DT, CT, DP, 1>(a, atoms_most, s);
  else
    launch_columns<DT, CT, DP, 2>(a, atoms_most, s);
  return pl_launch_status("pl_tree_attention");
}

// Columns of a launch: as many as there are workers for, at least one token's.
constexpr int kColumnsMax = kColTilesMax * kCols;

template <int DT, int CT>
int launch(int32_t dtype, int32_t cache_dtype, tree_args a, int64_t atoms_most, hipStream_t s) {
  const int toks = kColumnsMax / a.group;
  for (a.tok0 = 0; a.tok0 < a.row_len; a.tok0 += toks) {
    a.toks = a.row_len - a.tok0 < toks ? a.row_len - a.tok0 : toks;
    const int rc = a.dim <= 64    ? launch_dim<DT, CT, 64>(dtype, cache_dtype, a, atoms_most, s)
                   : a.dim <= 128 ? launch_dim<DT, CT, 128>(dtype, cache_dtype, a, atoms_most, s)
                                  : launch_dim<DT, CT, 256>(dtype, cache_dtype, a, atoms_most, s);
    if (rc) return rc;
  }
  return PL_OK;
}

}  // namespace

static_assert(PL_ATTENTION_COUNTER_INTS == kWorkersMax * kCounterStride, "one counter per workgroup");

extern "C" int64_t pl_tree_attention_workspace_bytes(int32_t dim, int32_t columns) {
  if (dim < 1 || dim > kHeadDimMax || columns < 0) return 0;
  // two parts of a worker: of up to kWorkersMax workers of 32 columns each (16 of large heads), or, of
  // 16-bit models, of one on a CU of 256 (128)
  const int dp = dim <= 64 ? 64 : dim <= 128 ? 128 : 256;
  const int64_t sixteens = columns <= narrow_columns(dp) ? 2ll * kWorkersMax * (dp == 256 ? 1 : 2) : 2ll * kCus * wide_columns(dp) / kCols;
  return sixteens * part_floats(dp) * (int64_t)sizeof(float);
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
  if (heads / kv_heads > kColumnsMax) {
    pl_set_error("%s: at most %d query heads to a key head (got %d)", what, kColumnsMax, heads / kv_heads);
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
  const int64_t all_columns = (int64_t)row_len * (heads / kv_heads);
  // (fp32 has the kernel for few columns alone)
  const int32_t columns = dtype == PL_F32 ? 1 : (int32_t)(all_columns < kColumnsMax ? all_columns : kColumnsMax);
  const int64_t need = pl_tree_attention_workspace_bytes(dim, columns);
  if (!workspace || workspace_bytes < need || !counters || counter_ints < PL_ATTENTION_COUNTER_INTS) {
    pl_set_error("%s: workspace of %lld bytes and %lld counters, %lld and %d needed", what, (long long)workspace_bytes,
                 (long long)counter_ints, (long long)need, PL_ATTENTION_COUNTER_INTS);
    return PL_ERR_ARG;
  }
  if (!on_a_line(workspace)) {
    pl_set_error("%s: the workspace must begin at whole %d bytes", what, kLine);
    return PL_ERR_ALIGN;
  }
  tree_args a;
  a.q = q, a.q_row = q_strides[0], a.q_token = q_strides[1], a.q_head = q_strides[2];
  a.key = {const_cast<void*>(key_cache), key_strides[0], key_strides[1], key_strides[2]};
  a.value = {const_cast<void*>(value_cache), value_strides[0], value_strides[1], value_strides[2]};
  a.table = {page_table, table_ld, max_pages, num_pages, pl_log2_exact(page_size)};
  a.past = past_lens, a.seq_lens = seq_lens, a.visible = visible, a.visible_row = visible_row;
  a.visible_token = visible_token, a.depths = visible ? depths : nullptr, a.depths_row = depths_row;
  a.k_scale = k_scale, a.v_scale = v_scale, a.out = out, a.scale = scale, a.rows = rows, a.row_len = row_len;
  a.heads = heads, a.kv_heads = kv_heads, a.dim = dim, a.window = window, a.group = heads / kv_heads, a.per_group = 1.f / (float)a.group;
  a.parts = static_cast<float*>(workspace), a.counters = counters;
  // lines are marked as read once where a pool of pages is too large for the last cache
  a.once = 2ll * num_pages * ((int64_t)kv_heads * dim * page_size) * pl_cache_elem_size(cache_dtype) > (256 << 20);
  // atoms at most: every row as long as its pages or its window allow
  int64_t longest = (int64_t)max_pages * page_size;
  if (window > 0 && longest > (int64_t)window + row_len + 31) longest = (int64_t)window + row_len + 31;
  const int64_t atom = 32 * kWaves, per_pair = longest > atom ? (longest + atom - 1) / atom : 1;
  const int64_t pairs = (int64_t)rows * kv_heads;
  // token and atom numbers are 32-bit, stages past a row's end and a run past the last one included
  if ((int64_t)max_pages * page_size > INT32_MAX - 8 * atom || pairs > (INT32_MAX - kWorkersMax) / per_pair) {
    pl_set_error("%s: %lld rows and key heads of up to %lld tokens are too many", what, (long long)pairs,
                 (long long)longest);
    return PL_ERR_LIMIT;
  }
  const int64_t atoms_most = pairs * per_pair;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (cache_dtype == PL_F8E4M3)
    return dtype == PL_BF16 ? launch<PL_BF16, PL_F8E4M3>(dtype, cache_dtype, a, atoms_most, s)
                            : launch<PL_F16, PL_F8E4M3>(dtype, cache_dtype, a, atoms_most, s);
  if (dtype == PL_F32) return launch<PL_F32, PL_F32>(dtype, cache_dtype, a, atoms_most, s);
  return dtype == PL_BF16 ? launch<PL_BF16, PL_BF16>(dtype, cache_dtype, a, atoms_most, s)
                          : launch<PL_F16, PL_F16>(dtype, cache_dtype, a, atoms_most, s);
}
