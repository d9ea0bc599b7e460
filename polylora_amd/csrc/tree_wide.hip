// Attention of drafted tokens where the row's tokens times the heads of a key head make
// many columns.
//
// Products bound it then, not memory: each key and value takes part in as many of them
// as there are columns.  A workgroup of eight waves keeps up to 256 columns (128 for heads
// above 128 elements) and brings keys and values to LDS once for all of them, 32 KB at
// a time, one stage read and three on their way (two of 64 KB took the same), by loads
// that go past the registers.  Two waves of a SIMD take turns at its matrix and its
// vector unit.  Waves
// stand side by side over the columns, and where those are few, behind one
// another over the tokens of a stage: `across` times 32 (16) columns, and the
// stage's 32-token units dealt out to the waves of a column in turn.
//
// In LDS a row of pieces of 16 bytes is turned by its number (its pieces' places XORed), so
// that 16 rows' pieces of one place, which the keys' product asks for, lie in 16
// different quarters of the banks.
//
// Measured, bf16, 32 query heads over 8 of 128: 64 drafts of 16 rows over 8192 tokens 195 to 250 us
// by the rows' lengths (49 us of products at the rate of a large one, 65 of bytes);
// of one row 57.  With weights in two parts of 16 bits a unit of 32 tokens by 32 columns took a wave about
// 2100 cycles, nearly the sum of its 832 of products and 950 of weights: the two waves of a SIMD
// overlap little.  The third part, which holds the rest of the weight (kWeightParts), adds 288 of products
// and took 64 rows of 32 drafts over 4096 tokens from 240 to 267 us; one part alone took a fifth less than two.
#include "pl_tree.h"

namespace {

constexpr int kWideThreads = kWideWaves * 64;
constexpr int kStageBytes = 32 << 10;
constexpr int kBuffers = 4;  // one is read, three are on their way

template <int DT, int CT, int DP>
struct wide : shape<DT, CT, DP> {
  typedef shape<DT, CT, DP> S;
  static constexpr int C = DP == 256 ? 1 : 2;
  static constexpr int kRow = DP * S::kCsize;   // bytes of a token in LDS
  static constexpr int kSlots = kRow / 16;      // its pieces
  static constexpr int kFit = kStageBytes / (2 * 32 * kRow);
  static constexpr int kUnits = kFit < 4 ? kFit : 4;  // of a stage, 32 tokens each
  static constexpr int kSide = kUnits * 32 * kRow;    // bytes of a stage's keys, then as many of values
  static constexpr int kChunks = kSide / 1024;        // loads of a wave: 64 lanes, 16 bytes each
  static constexpr int kChunkRows = 1024 / kRow;
  static constexpr int kJoin = kWideWaves * kCols * (DP + 4) * 4;
  static constexpr int kOwn = kChunks / kWideWaves;   // a wave's, of keys and again of values
  static constexpr int kLds = kBuffers * 2 * kSide > kJoin ? kBuffers * 2 * kSide : kJoin;
  // What a row's pieces are turned by.
  static __device__ __forceinline__ int turn(int row) {
    return kSlots >= 16 ? row & 15 : kSlots == 8 ? row >> 1 & 7 : row >> 2 & 3;
  }
};

__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}
// 16 bytes to a lane, from p + lane_off to LDS at `to` + 16 * lane.  The wait for it is the
// caller's, before the barrier behind which the stage is read.  (The compiler sets m0 where it wants it
// and keeps nothing else there, but may take it to be still what it set: so it is named, and the
// warning about reserved registers is off.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_to_lds(uint32_t to, uintptr_t p, uint32_t bytes, uint32_t lane_off) {
  const pl_u32x4 r = {(uint32_t)uniform((int)(uint32_t)p), (uint32_t)uniform((int)(p >> 32)), (uint32_t)uniform((int)bytes),
                      0x00027000u};
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(uniform((int)to)), "v"(lane_off), "s"(r)
               : "memory", "m0");
}
#pragma clang diagnostic pop

// Joins n parts of columns [in0, in1) (numbers of sixteens: the first part's, and from the
// second on first + step * part) and puts out what comes of them.  A thread has ITEMS
// places in hand, BATCH parts of each at a time: parts come from where every XCD
// sees them, and what counts is how many are on their way.
template <typename T, int DP, bool FULL, int ITEMS, int BATCH>
__device__ __forceinline__ void join_columns(const tree_args& a, pl_buffer parts, int first, int others, int step, int n,
                                             int row, int col0, int in0, int in1, int live, int hk, float v_scale,
                                             int threads) {
  typedef part_layout<DP> P;
  const int items = (in1 - in0) * (DP / 4);
  for (int i0 = (int)threadIdx.x; i0 < items; i0 += ITEMS * threads) {
    float top[ITEMS], sum[ITEMS];
    pl_f32x4 y[ITEMS];
#pragma unroll
    for (int s = 0; s < ITEMS; ++s) top[s] = -INFINITY, sum[s] = 0.f, y[s] = pl_f32x4{0.f, 0.f, 0.f, 0.f};
    for (int k0 = 0; k0 < n; k0 += BATCH) {
      pl_f32x4 x[ITEMS][BATCH];
      pl_f32x2 ml[ITEMS][BATCH];
#pragma unroll
      for (int s = 0; s < ITEMS; ++s)
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
          const int i = min(i0 + s * threads, items - 1), in = in0 + i / (DP / 4), d = i % (DP / 4) * 4;
          const int k = min(k0 + j, n - 1);  // the last again, with no weight
          const uint32_t part = (uint32_t)((k ? others + step * k : first) + in / kCols) * P::kBytes;
          x[s][j] = __builtin_bit_cast(
              pl_f32x4, __builtin_amdgcn_raw_buffer_load_b128(parts, part + P::at(in % kCols, d), 0, kAgentScope));
          ml[s][j] = __builtin_bit_cast(
              pl_f32x2, __builtin_amdgcn_raw_buffer_load_b64(parts, part + P::sums(in % kCols), 0, kAgentScope));
        }
#pragma unroll
      for (int s = 0; s < ITEMS; ++s) {
        float high = top[s];
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
          ml[s][j].x = k0 + j < n ? ml[s][j].x : -INFINITY;
          high = fmaxf(high, ml[s][j].x);
        }
        const float ref = high == -INFINITY ? 0.f : high, keep = exp2_fast(top[s] - ref);
        sum[s] *= keep, y[s] *= keep, top[s] = high;
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
          const float f = exp2_fast(ml[s][j].x - ref);
          sum[s] += f * ml[s][j].y, y[s] += f * x[s][j];
        }
      }
    }
#pragma unroll
    for (int s = 0; s < ITEMS; ++s) {
      const int i = i0 + s * threads;
      if (i < items)
        put_output<T, FULL>(a, row, col0, in0 + i / (DP / 4), live, hk, i % (DP / 4) * 4, y[s], sum[s], v_scale);
    }
  }
}

// The parts of pairs that are cut into many: a workgroup to every four columns of a pair,
// where one that arrives last would have all of them to itself (1 x 16 drafts over
// 131072 tokens, 32 parts to a pair: 7 us; 26 with sixteens and two parts at a time).
constexpr int kJoinThreads = 128, kJoinColumns = 4;
template <int DT, int CT, int DP, bool FULL>
__global__ __launch_bounds__(kJoinThreads) void pl_tree_join_kernel(tree_args a) {
  typedef wide<DT, CT, DP> S;
  typedef typename pl_traits<DT>::T T;
  constexpr int kSixteens = kWideWaves * S::C, kShares = wide_columns(DP) / kJoinColumns;
  const int lane = (int)threadIdx.x & 63;
  const int share = (int)blockIdx.x % kShares, ct = (int)blockIdx.x / kShares % a.col_tiles;
  const int pair = (int)blockIdx.x / kShares / a.col_tiles, row = pair / a.kv_heads, hk = pair % a.kv_heads;
  const int col0 = ct * wide_columns(DP), cols = min(wide_columns(DP), a.toks * a.group - col0);
  const int in0 = share * kJoinColumns, in1 = min(in0 + kJoinColumns, cols);
  if (in0 >= in1) return;
  // the deal, and the atoms before this row
  const tree_run run = find_run<S::kAtom, S::kAtom / 128>(a, 0, lane);
  if (run.whole_pairs) return;
  int before = 0;
  for (int b = lane; b < row; b += 64) before += span_of<S::kAtom>(a, a.past[b], a.seq_lens ? a.seq_lens[b] : a.row_len).atoms;
  before = __builtin_amdgcn_readlane(scan_sum(before), 63) * a.kv_heads;
  const tree_span r = span_of<S::kAtom>(a, a.past[row], a.seq_lens ? a.seq_lens[row] : a.row_len);
  const int pair_start = before + hk * r.atoms;
  const int w0 = pair_start / run.per, w1 = (pair_start + r.atoms - 1) / run.per;
  if (w0 == w1) return;  // in one piece: its worker has put it out
  const int live = max(0, min(cols, (min(r.n, a.tok0 + a.toks) - a.tok0) * a.group - col0));
  const int slot1 = 2 * (w0 * a.col_tiles + ct), slot0 = slot1 + (w0 * run.per == pair_start ? 0 : 1);
  join_columns<T, DP, FULL, 1, 8>(a, part_layout<DP>::all(a.parts, 2u * kWorkersMax / 2 * kSixteens), slot0 * kSixteens,
                            slot1 * kSixteens, 2 * a.col_tiles * kSixteens, w1 - w0 + 1, row, col0, in0, in1, live, hk,
                            CT == PL_F8E4M3 ? a.v_scale[hk] : 1.f, kJoinThreads);
}

template <int DT, int CT, int DP, bool FULL>
__global__ __launch_bounds__(kWideThreads, 2) void pl_tree_wide_kernel(tree_args a, int across, int join_later) {
  typedef wide<DT, CT, DP> S;
  typedef typename pl_traits<DT>::T T;
  constexpr int C = S::C, kParts = kWeightParts<DT>;
  constexpr float kLift = DT == PL_F16 ? 15.f - kSlack : 0.f;
  __shared__ __attribute__((aligned(1024))) uint8_t s_mem[S::kLds];
  __shared__ float s_m[kWideWaves][kCols], s_l[kWideWaves][kCols];
  __shared__ int s_held[kBuffers][2 * S::kUnits];
  __shared__ int s_last;
  const int tid = (int)threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int li = lane & 15, lg = lane >> 4;
  const int wc = wave % across, wt = wave / across, behind = kWideWaves / across;
  // Of a SIMD's two waves one goes first, so that they are not both at their products or
  // both at their weights (16 drafts of 16 rows over 8192, as it was then in this kernel: 107 ->
  // 101 us; 64 drafts 230 -> 227).
  if (wave < kWideWaves / 2) __builtin_amdgcn_s_setprio(1);
  const tree_worker me = worker_of(a);
  const int ct = me.ct, slice = me.slice;
  const tree_run run = find_run<S::kAtom, S::kAtom / 128>(a, slice, lane);
  const int from = run.from, to = run.to, per = run.per;
  const bool whole_pairs = run.whole_pairs;
  if (from >= run.total) return;
  int row = run.row, row_start = run.row_start, row_past = run.row_past, row_new = run.row_new, at = from;
  bool skip = whole_pairs;  // to the first pair that starts in the run

  if constexpr (!FULL) {
    // pieces past the head's end are never loaded
    for (int i = tid; i < S::kLds / 16; i += kWideThreads)
      reinterpret_cast<shared_u32x4*>(s_mem)[i] = pl_u32x4{0, 0, 0, 0};
    __syncthreads();
  }
  // where this lane reads: its key of 16, a piece to each load, and its share of four values
  uint32_t key_at[S::kKeyLoads], value_at[4][S::kPieces];
#pragma unroll
  for (int n = 0; n < S::kKeyLoads; ++n) key_at[n] = li * S::kRow + ((n * 4 + lg) ^ S::turn(li)) * 16;
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int n = 0; n < S::kPieces; ++n) {
      const int token = 4 * lg + j, byte = S::value_at(li, n) * S::kCsize;
      value_at[j][n] = S::kSide + token * S::kRow + ((byte / 16) ^ S::turn(token)) * 16 + byte % 16;
    }

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
    // this worker's columns, and those of tokens that count; this wave's are sixteens wc and wc + across
    const int col0 = ct * wide_columns(DP), cols = min(across * C * kCols, a.toks * a.group - col0);
    const int live = max(0, min(cols, (min(r.n, a.tok0 + a.toks) - a.tok0) * a.group - col0));

    pl_f32x4 o[C][S::V];
    float m[C];
    pl_f32x4 l[C];
    int t[C], first[C], all_from = 0;
    pl_u32x4 q[C][S::kSteps];
    const float signed_scale = a.scale * 1.44269504088896f * (CT == PL_F8E4M3 ? as_scalar(a.k_scale)[hk] : 1.f);
    const float scale2 = fmaxf(fabsf(signed_scale), 1.17549435e-38f);
    const uint32_t flip = signed_scale < 0.f ? 0x80008000u : 0u;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      m[c] = -INFINITY, l[c] = pl_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < S::V; ++i) o[c][i] = pl_f32x4{0.f, 0.f, 0.f, 0.f};
      const int in = (wc + c * across) * kCols + li;
      const column_place at = place_of(a, col0 + in, hk);
      t[c] = in < live ? at.token : -1;
      first[c] = first_seen(a, r, row, t[c]);
      all_from = max(all_from, first[c]);
#pragma unroll
      for (int n = 0; n < S::kSteps; ++n) {
        const int d = CT == PL_F8E4M3 ? key_piece<CT>(n / 2, lg, S::E) + (n % 2) * 8 : key_piece<CT>(n, lg, S::E);
        q[c][n] = pl_u32x4{0, 0, 0, 0};
        // rows of q have the alignment of their elements alone
        if (in < live && (FULL || d < a.dim))
          __builtin_memcpy(&q[c][n], (const T*)a.q + row * a.q_row + at.token * a.q_token + at.head * a.q_head + d, 16);
        q[c][n] ^= flip;
      }
    }
    all_from = a.window > 0 ? __builtin_amdgcn_readlane(scan_max(all_from), 63) : 0;

    // a line's last column sees the most; no column that counts, no token
    const int last_t = uniform(place_of(a, max(0, col0 + live - 1), hk).token);
    const int seen = a.visible ? r.len : (int)min((int64_t)r.len, (int64_t)r.past + last_t + 1);
    const int begin = r.base + first_atom * S::kAtom;
    const int end = live > 0 ? min(seen, r.base + last_atom * S::kAtom) : 0;
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

    // One stage's keys and values, a kilobyte at a time; 16 tokens share a page.  Its
    // pages are asked for a stage ahead.  What is not there is asked for with no bytes, so
    // that every stage is as many loads.
    int ids[S::kOwn];
    auto look_up = [&](int base, int (&ids)[S::kOwn]) __attribute__((always_inline)) {
#pragma unroll
      for (int k = 0; k < S::kOwn; ++k) {
        const int token = base + ((wave + k * kWideWaves) * S::kChunkRows & ~15);
        // no look-up past the end: the table's row may end there
        ids[k] = token < end ? w.pages[token >> w.shift] : -1;
      }
    };
    auto load_stage = [&](int buffer, int base, const int(&ids)[S::kOwn]) __attribute__((always_inline)) {
      const uint32_t lds = lds_address(s_mem) + buffer * 2 * S::kSide;
#pragma unroll
      for (int k = 0; k < S::kOwn; ++k) {
        const int chunk = wave + k * kWideWaves, row0 = chunk * S::kChunkRows;
        const int in = (row0 & 15) + lane / S::kSlots;  // of the 16 tokens
        const int piece = lane % S::kSlots ^ S::turn(in);
        const bool held = ids[k] >= 0 && ids[k] < w.num_pages;
        const int64_t page = held ? ids[k] : 0;
        const uint32_t slot = (uint32_t)(base + (row0 & ~15)) & ((1u << w.shift) - 1);
        if (row0 % 16 == 0 && lane == 0) s_held[buffer][row0 / 16] = held;
        if (FULL || piece * 16 < a.dim * S::kCsize) {
          load_to_lds(lds + chunk * 1024, w.key + page * w.key_page + (uint64_t)slot * w.key_slot, held ? key_span : 0,
                      in * w.key_slot + piece * 16);
          load_to_lds(lds + S::kSide + chunk * 1024, w.value + page * w.value_page + (uint64_t)slot * w.value_slot,
                      held ? value_span : 0, in * w.value_slot + piece * 16);
        }
      }
    };

    bool nonfinite = false;  // values of a mixed unit were infinities or NaN
    uint32_t all_held = 0;   // which 16 tokens of the stage lie on pages that the table holds
    // A unit: 32 tokens of the stage.
    auto unit = [&](int buffer, int u, int tile) __attribute__((always_inline)) {
      const uint8_t* mem = s_mem + buffer * 2 * S::kSide + u * 32 * S::kRow;
      pl_f32x4 s[2][C];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int c = 0; c < C; ++c) s[h][c] = pl_f32x4{0.f, 0.f, 0.f, 0.f};
      // all keys of a step asked for before the first product: a wave has little else to
      // wait behind
      constexpr int kAhead = S::kKeyLoads < 4 ? S::kKeyLoads : 4;
#pragma unroll
      for (int n0 = 0; n0 < S::kKeyLoads; n0 += kAhead) {
        pl_u32x4 keys[kAhead][2];
#pragma unroll
        for (int n = 0; n < kAhead; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            keys[n][h] = *reinterpret_cast<const shared_u32x4*>(mem + h * 16 * S::kRow + key_at[n0 + n]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < kAhead; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const pl_u32x4 k = keys[n][h];
            if constexpr (CT == PL_F8E4M3) {
              const pl_u32x4 x = {widen<DT, false>(k.x), widen<DT, true>(k.x), widen<DT, false>(k.y),
                                  widen<DT, true>(k.y)};
              const pl_u32x4 y = {widen<DT, false>(k.z), widen<DT, true>(k.z), widen<DT, false>(k.w),
                                  widen<DT, true>(k.w)};
#pragma unroll
              for (int c = 0; c < C; ++c) s[h][c] = pl_mfma_chunk<DT>(x, q[c][2 * (n0 + n)], s[h][c]);
#pragma unroll
              for (int c = 0; c < C; ++c) s[h][c] = pl_mfma_chunk<DT>(y, q[c][2 * (n0 + n) + 1], s[h][c]);
            } else {
#pragma unroll
              for (int c = 0; c < C; ++c) s[h][c] = pl_mfma_chunk<DT>(k, q[c][n0 + n], s[h][c]);
            }
          }
      }
      uint32_t v[S::kTokens][S::kVWords];
#pragma unroll
      for (int j = 0; j < S::kTokens; ++j)
#pragma unroll
        for (int n = 0; n < S::kPieces; ++n)
          __builtin_memcpy(v[j] + n * (S::kVWords / S::kPieces),
                           __builtin_assume_aligned(mem + j / 4 * 16 * S::kRow + value_at[j % 4][n],
                                                    S::kPiece * S::kCsize),
                           S::kPiece * S::kCsize);
      float p[C][S::kTokens];
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int j = 0; j < S::kTokens; ++j) p[c][j] = s[j / 4][c][j % 4];
      const bool held[2] = {(all_held >> 2 * u & 1) != 0, (all_held >> 2 * u & 2) != 0};
      if (__builtin_expect(!(tile >= all_from && tile + 32 <= min(r.past, r.len) && held[0] && held[1]), 0))
        nonfinite |= mask_tile<DT, CT, DP, C>(a, r, row, t, first, tile, held, lane, p, v);
      rescale<S::kTokens, S::V, C>(p, scale2, m, l, o);
      pl_u32x4 part[C][kParts];
#pragma unroll
      for (int c = 0; c < C; ++c) {
        // nothing alive yet: any finite reference gives weights of 0
        const float ref = (m[c] == -INFINITY ? 0.f : m[c]) - kLift;
#pragma unroll
        for (int j = 0; j < S::kTokens; ++j) p[c][j] = exp2_fast(fmaf(p[c][j], scale2, -ref));
        weight_parts<DT>(p[c], part[c]);
      }
      add_values<DT, CT, DP, C>(v, part, o, l);
    };

    constexpr int kStage = S::kUnits * 32;
    if (begin < end) {
      int first_ids[kBuffers - 1][S::kOwn];
#pragma unroll
      for (int i = 0; i < kBuffers - 1; ++i) look_up(begin + i * kStage, first_ids[i]);
      look_up(begin + (kBuffers - 1) * kStage, ids);
#pragma unroll
      for (int i = 0; i < kBuffers - 1; ++i) load_stage(i, begin + i * kStage, first_ids[i]);
    }
    int buffer = 0;
    for (int base = begin; base < end; base += kStage, buffer = (buffer + 1) % kBuffers) {
      // this stage is there (all but the two behind it), and nobody reads the one before it any more
      constexpr int kBehind = (kBuffers - 2) * 2 * S::kOwn;
      __builtin_amdgcn_s_waitcnt(0x0F70 | (kBehind & 15) | (kBehind >> 4) << 14);  // vmcnt
      __syncthreads();
      load_stage((buffer + kBuffers - 1) % kBuffers, base + (kBuffers - 1) * kStage, ids);
      look_up(base + kBuffers * kStage, ids);
      all_held = (uint32_t)__ballot(lane < 2 * S::kUnits && s_held[buffer][min(lane, 2 * S::kUnits - 1)]);
      for (int u = wt; u < S::kUnits && base + u * 32 < end; u += behind)
        if (wc * kCols < live) unit(buffer, u, base + u * 32);
    }
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): the join writes where loads are on their way
    if (__builtin_expect(nonfinite, 0))
      for (int base = begin; base < end; base += kStage)
        for (int u = wt; u < S::kUnits && base + u * 32 < end; u += behind) {
          const int tile = base + u * 32;
          const tile_place<2> here = place_tile<2>(w, tile);
          if (!(tile >= all_from && tile + 32 <= min(r.past, r.len) && here.held[0] && here.held[1]))
            add_nonfinite<DT, CT, DP, C, FULL>(a, r, row, t, first, tile, here, w.value_slot, lane, o);
        }

    // join the waves behind one another, 16 columns of each at a time
    const float v_scale = CT == PL_F8E4M3 ? as_scalar(a.v_scale)[hk] : 1.f;
    const bool complete = first_atom == 0 && last_atom == r.atoms;
    typedef part_layout<DP> P;
    constexpr int kSixteens = kWideWaves * C;
    const int slot = 2 * (slice * a.col_tiles + ct) + (at == from ? 0 : 1);
    const pl_buffer parts = P::all(a.parts, 2u * kWorkersMax / 2 * kSixteens);
    float* s_o = reinterpret_cast<float*>(s_mem);
    constexpr int kPitch = DP + 4;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      __syncthreads();
      if (lg == 0) s_m[wave][li] = m[c], s_l[wave][li] = l[c].x;
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int i = 0; i < S::V; i += 4)
          *reinterpret_cast<pl_f32x4*>(s_o + (wave * kCols + li) * kPitch +
                                       S::value_at(4 * lg + e, i / S::kPiece) + i % S::kPiece) =
              pl_f32x4{o[c][i][e], o[c][i + 1][e], o[c][i + 2][e], o[c][i + 3][e]};
      __syncthreads();
      for (int i = tid; i < across * kCols * (DP / 4); i += kWideThreads) {
        const int col = i / (DP / 4), d = i % (DP / 4) * 4, w0 = col / kCols;
        float top = -INFINITY, sum = 0.f;
        pl_f32x4 x = {0.f, 0.f, 0.f, 0.f};
        for (int k = w0; k < kWideWaves; k += across) top = fmaxf(top, s_m[k][col % kCols]);
        const float ref = top == -INFINITY ? 0.f : top;
        for (int k = w0; k < kWideWaves; k += across) {
          const float f = exp2_fast(s_m[k][col % kCols] - ref);
          sum += f * s_l[k][col % kCols];
          x += f * *reinterpret_cast<const pl_f32x4*>(s_o + (k * kCols + col % kCols) * kPitch + d);
        }
        const int in = c * across * kCols + col;
        if (in >= cols) continue;
        if (complete)
          put_output<T, FULL>(a, row, col0, in, live, hk, d, x, sum, v_scale);
        else
          put_part<DP>(parts, slot * kSixteens, in, d, x, top, sum);
      }
    }
    if (!complete && !join_later) {
      const int w0 = pair_start / per, w1 = (pair_start + r.atoms - 1) / per;
      if (arrive_last(a.counters + (w0 * a.col_tiles + ct) * kCounterStride, w1 - w0, &s_last)) {
        // the first part is its workgroup's second when that workgroup began earlier
        const int slot1 = 2 * (w0 * a.col_tiles + ct), slot0 = slot1 + (w0 * per == pair_start ? 0 : 1);
        const int n = w1 - w0 + 1;
        join_columns<T, DP, FULL, 4, 2>(a, parts, slot0 * kSixteens, slot1 * kSixteens, 2 * a.col_tiles * kSixteens, n, row, col0,
                                  0, cols, live, hk, v_scale, kWideThreads);
      }
    }
    __syncthreads();  // the shared arrays are free again
    at = pair_start + last_atom;
    if constexpr (!FULL) {
      // the join wrote over pieces that are never loaded
      for (int i = tid; at < to && i < S::kLds / 16; i += kWideThreads)
        reinterpret_cast<shared_u32x4*>(s_mem)[i] = pl_u32x4{0, 0, 0, 0};
      __syncthreads();
    }
  }
}

// Slices to a pair above which parts are joined by a launch of their own, in many workgroups;
// up to it the last workgroup of a pair joins them, and saves the launch.  In us, always apart
// / from 2 / from 4 on (weights in two parts): 64 drafts of 16 rows over 8192 232 / 246 / 234, over 1024 69 / 69 / 65.5,
// 32 rows of 16 over 2000 89 / 78 / 78.
constexpr int kManyParts = 3;

template <int DT, int CT, int DP>
void launch_wide(tree_args a, int64_t atoms_most, hipStream_t s) {
  const int columns = a.toks * a.group, most = wide_columns(DP);
  a.col_tiles = (columns + most - 1) / most;
  a.slices = slices_of(atoms_most, kCus, a.col_tiles);
  int across = 1;
  while (across < kWideWaves && across * kCols * wide<DT, CT, DP>::C < columns) across *= 2;
  const dim3 grid((unsigned)(a.slices * a.col_tiles));
  const int64_t pairs = (int64_t)a.rows * a.kv_heads;
  const int later = a.slices > kManyParts * pairs;
  const dim3 joins((unsigned)(later ? pairs * a.col_tiles * (wide_columns(DP) / kJoinColumns) : 0));
  if (a.dim == DP) {
    pl_tree_wide_kernel<DT, CT, DP, true><<<grid, kWideThreads, 0, s>>>(a, across, later);
    if (later) pl_tree_join_kernel<DT, CT, DP, true><<<joins, kJoinThreads, 0, s>>>(a);
  } else {
    pl_tree_wide_kernel<DT, CT, DP, false><<<grid, kWideThreads, 0, s>>>(a, across, later);
    if (later) pl_tree_join_kernel<DT, CT, DP, false><<<joins, kJoinThreads, 0, s>>>(a);
  }
}

template <int DT, int CT>
int launch(const tree_args& a, int64_t atoms_most, hipStream_t s) {
  if (a.dim <= 64)
    launch_wide<DT, CT, 64>(a, atoms_most, s);
  else if (a.dim <= 128)
    launch_wide<DT, CT, 128>(a, atoms_most, s);
  else
    launch_wide<DT, CT, 256>(a, atoms_most, s);
  return pl_launch_status("pl_tree_attention");
}

}  // namespace

int pl_tree_wide(int32_t dtype, int32_t cache_dtype, const tree_args& a, int64_t atoms_most, hipStream_t s) {
  if (cache_dtype == PL_F8E4M3)
    return dtype == PL_BF16 ? launch<PL_BF16, PL_F8E4M3>(a, atoms_most, s) : launch<PL_F16, PL_F8E4M3>(a, atoms_most, s);
  return dtype == PL_BF16 ? launch<PL_BF16, PL_BF16>(a, atoms_most, s) : launch<PL_F16, PL_F16>(a, atoms_most, s);
}
