// Attention of one new token per row over a paged key-value cache.
//
// With s_j = scale * q . k_j over the tokens j of a row,
//   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),   m = max_j s_j,
// in one pass over keys and values: a running maximum m, sum l and unscaled
// output o, all fp32; a larger maximum rescales l and o by exp(m_old - m), and
// two partial results (m, l, o) of disjoint tokens join by the same rule.
//
// Each key and value element is read once and takes 2 * heads / kv_heads
// operations a head, a few per byte: memory bounds it.  What carries it is
// that every wave has whole tiles of loads in flight and nothing is staged:
// keys and values go from their pages straight into the registers that feed
// the matrix instructions.
//
// A wave takes tiles of 32 tokens (16 in fp32) of one (row, key head) and the
// up to 16 query heads that share it, one per column of a 16x16 matrix
// product; lane l stands for column l % 16 and lane group l / 16.
//   S^T = K Q^T   lane (i, g) supplies 16-byte pieces of token i's key and of
//                 query i; it gets the scores of query i with tokens 4g .. 4g+3
//                 of each 16.
//   O^T = V^T P^T the contraction over tokens may take them in any order that
//                 both operands share, so each lane keeps the tokens whose
//                 scores it got: the weights never leave their lane, and the
//                 lane reads those tokens' values, a sixteenth of each, and
//                 pairs them up by byte permutes.  It gets the outputs of
//                 query i, so the maximum, the sum and the rescaling of a query
//                 all stay in the lanes of its column.
// Weights go into the product as sums of 16-bit numbers, a product more for each
// on matrix units that have little else to do: three bf16 are the fp32 weight
// itself, two fp16 keep 2^-21 of it, and the output keeps the error of its own
// rounding (two bf16, 2^-15 of a weight, put 8 times as many outputs on the other
// side of theirs, 0.33 % of them, for 0.5 us of 110 over 256 rows to 1024 tokens
// and 0.7 of 21 over 64 of 512).  fp16 ends at 2^-24, so its weights are taken
// 2^15 times as large, to 32768 for the highest score (l and o alike, so the
// factor goes out in o / l), and end at 2^-39 of the largest; without it tokens
// 17.3 and more below the highest score counted in l and not in o.
//
// Work is split by tokens: the launch is a fixed number of workgroups, and the
// batch's atoms (kAtom tokens of one row and key head) are dealt out in equal
// runs, found from the lengths on the device, so no length is needed on the
// host and ragged batches come out even (deal below says how runs are taken).
// Where runs end inside a (row, key head), each leaves (m, l, o) in the
// workspace, and the workgroup that arrives last on the pair's counter joins
// the parts in order (the same bits whichever arrives last).
#include "pl_paged.h"

namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr int kCols = 16;  // query heads of a workgroup's products

// Workgroups of a launch: two on each CU, of which a batch of many tokens takes
// one.  A CU's waves are served oldest first, so its workgroups end one after
// the other, and the memory is as busy with the fewer of them: with three,
// two and one on a CU, a row of 131072 tokens takes 103, 96 and 91 us, 256 rows
// of up to 1024 121, 118 and 115; 64 rows of up to 512, starting and ending
// more than reading, 22, 22 and 25; fp32, 37 x 12 windows of 500, 42, 34 and 39;
// 51 rows of up to 18000 over an 8-bit cache of 80 elements, 75 with two and 83
// with one.
constexpr int kCus = 256;
constexpr int kWorkersMax = 2 * kCus;
constexpr int kManyAtoms = 8 * kCus;
constexpr int kCounterStride = 16;  // int32s: 64 bytes for each counter

template <int DT, int CT, int DP>
struct shape {
  static constexpr int E = pl_traits<DT>::E;         // elements of a 16-byte piece
  static constexpr int kSubs = DT == PL_F32 ? 1 : 2; // 16-token parts of a tile
  static constexpr int kTile = 16 * kSubs;
  static constexpr int kAtom = 32 * kWaves;
  static constexpr int kSteps = DP / (4 * E);        // products of 4 pieces along a key
  static constexpr int kCsize = CT == PL_F8E4M3 ? 1 : DT == PL_F32 ? 4 : 2;
  static constexpr int kKeyLoads = DP * kCsize / 64; // 16-byte loads of a lane per 16 keys
  static constexpr int V = DP / 16;                  // value elements of a lane per token
  static constexpr int kVWords = V * kCsize / 4;
  // Waves of a SIMD that the compiler is to leave registers for: schedules
  // for fewer were slower (fp32, 64 x 12 x 2048 tokens: 161 -> 169 us).
  static constexpr int kWavesPerSimd = DP <= 128 ? 3 : 2;
  // They come in pieces of at most 16 bytes, 16 lanes' pieces side by side.
  static constexpr int kPiece = V * kCsize <= 16 ? V : 16 / kCsize;
  static constexpr int kPieces = V / kPiece;
  static __device__ __forceinline__ int value_at(int lane, int piece) {
    return (piece * 16 + lane) * kPiece;
  }
  static constexpr int kTokens = 4 * kSubs;          // tokens of a lane per tile
  // Queries in LDS where keys, values and outputs fill the registers (heads of
  // 144 to 240 elements spill a few all the same, 20 to 96 bytes a thread).
  static constexpr bool kQueryLds = DP == 256 || DT == PL_F32;
  static constexpr int kParts = DT == PL_BF16 ? 3 : 2;  // 16-bit parts of a weight
  // log2 of what weights are multiplied by, that their 16-bit parts keep small ones.
  static constexpr float kLift = DT == PL_F16 ? 15.f : 0.f;
};
typedef pl_u32x4 __attribute__((may_alias)) shared_u32x4;
typedef uint32_t pl_u32x2 __attribute__((ext_vector_type(2)));
typedef float pl_f32x2 __attribute__((ext_vector_type(2)));

struct attend_args {
  const void* q;
  int64_t q_row, q_head;
  pl_cache_view key, value;
  pl_page_table table;
  const int32_t* lens;
  const float *k_scale, *v_scale;
  void* out;  // contiguous [rows][heads][dim]
  float* parts;
  int32_t* counters;
  float scale;
  int32_t rows, heads, kv_heads, dim, window, group, col_tiles;
};

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Sum (and, of values that are not negative, maximum) of a lane's and all lower
// lanes' values: shifts by 1, 2, 4 and 8 inside rows of 16, then each row's
// last lane into the rows above.  Lanes that a step does not write add 0.
template <int CTRL, int ROWS>
__device__ __forceinline__ int from_lower(int x) {
  return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int scan_sum(int x) {
  x += from_lower<0x111, 0xf>(x), x += from_lower<0x112, 0xf>(x);
  x += from_lower<0x114, 0xf>(x), x += from_lower<0x118, 0xf>(x);
  x += from_lower<0x142, 0xa>(x);
  return x + from_lower<0x143, 0xc>(x);
}
__device__ __forceinline__ int scan_max(int x) {
  x = max(x, from_lower<0x111, 0xf>(x)), x = max(x, from_lower<0x112, 0xf>(x));
  x = max(x, from_lower<0x114, 0xf>(x)), x = max(x, from_lower<0x118, 0xf>(x));
  x = max(x, from_lower<0x142, 0xa>(x));
  return max(x, from_lower<0x143, 0xc>(x));
}

// The largest of the four lanes of a column, and their sum.
__device__ __forceinline__ float column_max(float x) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float column_sum(float x) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Memory that a wave's lanes read through a buffer descriptor, all of it in
// scalar registers: `bytes` from `p`; reads past them give 0 and touch nothing.
typedef __amdgpu_buffer_rsrc_t pl_buffer;
__device__ __forceinline__ pl_buffer make_buffer(uintptr_t p, uint32_t bytes) {
  const uint32_t lo = (uint32_t)uniform((int)(uint32_t)p), hi = (uint32_t)uniform((int)(p >> 32));
  return __builtin_amdgcn_make_buffer_rsrc(
      reinterpret_cast<void*>((uintptr_t)lo | (uintptr_t)hi << 32), 0, uniform((int)bytes), 0x00027000);
}
// N words (1, 2 or 4) at lane_off + wave_off; STREAM marks lines as read once.
template <int N, bool STREAM>
__device__ __forceinline__ void load_words(pl_buffer r, uint32_t lane_off, uint32_t wave_off,
                                           uint32_t* w) {
  constexpr int kPolicy = STREAM ? 2 : 0;
  if constexpr (N == 4) {
    const auto x = __builtin_amdgcn_raw_buffer_load_b128(r, lane_off, wave_off, kPolicy);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = x[i];
  } else if constexpr (N == 2) {
    const auto x = __builtin_amdgcn_raw_buffer_load_b64(r, lane_off, wave_off, kPolicy);
    w[0] = x[0], w[1] = x[1];
  } else {
    static_assert(N == 1, "loads of 4, 8 or 16 bytes");
    w[0] = __builtin_amdgcn_raw_buffer_load_b32(r, lane_off, wave_off, kPolicy);
  }
}

// Two e4m3 values of a word as a pair of the model's 16-bit type (exact).
template <int DT, bool HIGH>
__device__ __forceinline__ uint32_t widen(uint32_t w) {
  if constexpr (DT == PL_BF16)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, HIGH));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, HIGH));
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  typedef typename pl_traits<DT>::T T;
  typedef T T2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, T2{(T)a, (T)b});
}
template <int DT>
__device__ __forceinline__ float unpack(uint32_t w, int half) {
  typedef typename pl_traits<DT>::T T;
  typedef T T2 __attribute__((ext_vector_type(2)));
  return (float)__builtin_bit_cast(T2, w)[half];
}

// The same, rounded towards 0.
template <int DT>
__device__ __forceinline__ uint32_t pack2_down(float a, float b) {
  if constexpr (DT == PL_BF16)
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302);
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
}
// Numbers that are not negative, raised to the type's smallest normal one (fp16:
// smallest of all) beside ones that are not 0 in `first`.
template <int DT>
__device__ __forceinline__ uint32_t at_least_smallest(uint32_t x, uint32_t first) {
  typedef uint16_t pair __attribute__((ext_vector_type(2)));
  constexpr uint16_t kSmallest = DT == PL_BF16 ? 0x80 : 1;
  const pair least = __builtin_elementwise_min(__builtin_bit_cast(pair, first), pair{kSmallest, kSmallest});
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(pair, x), least));
}

// First element of the 16-byte key piece that lane group g loads n-th.
template <int CT>
__device__ __forceinline__ int key_piece(int n, int g, int e) {
  return (n * 4 + g) * (CT == PL_F8E4M3 ? 16 : e);
}

// What a wave holds of one (row, key head): its queries, and m (in units of
// log2 e), l (this lane's tokens alone) and o of its tiles so far.
template <int DT, int CT, int DP>
struct wave_state {
  typedef shape<DT, CT, DP> S;
  pl_u32x4 q[S::kQueryLds ? 1 : S::kSteps];
  shared_u32x4* q_lds;  // this lane's pieces, 64 apart
  __device__ __forceinline__ pl_u32x4 query(int n) const {
    if constexpr (S::kQueryLds)
      return q_lds[n * 64];
    else
      return q[n];
  }
  pl_f32x4 o[S::V];
  float m, l;
};

// A row's page ids, read through the scalar cache: every lane wants the same.
typedef const __attribute__((address_space(4))) int32_t* scalar_i32;
typedef const __attribute__((address_space(4))) float* scalar_f32;
__device__ __forceinline__ scalar_i32 as_scalar(const int32_t* p) {
  return (scalar_i32)(reinterpret_cast<uintptr_t>(p));
}
__device__ __forceinline__ scalar_f32 as_scalar(const float* p) {
  return (scalar_f32)(reinterpret_cast<uintptr_t>(p));
}

// What the walk over one (row, key head) needs; all of it is the wave's.
struct walk {
  uintptr_t key, value;  // the key head's
  scalar_i32 pages;
  int64_t key_page, value_page;  // bytes
  uint32_t key_slot, value_slot;
  int end, shift, num_pages;
};

// Where a tile's keys and values lie, for each 16 tokens of it (16 tokens from
// a multiple of 16 share a page).  Tokens past the walk's end and on pages that
// the table does not hold have no bytes: reading them gives 0.
template <int SUBS>
struct tile_place {
  uintptr_t key[SUBS], value[SUBS];
  bool held[SUBS];
};
template <int SUBS>
__device__ __forceinline__ tile_place<SUBS> place_tile(const walk& w, int t) {
  tile_place<SUBS> r;
#pragma unroll
  for (int u = 0; u < SUBS; ++u) {
    const int tu = t + 16 * u;
    // no look-up past the end: the table's row may end there
    const int id = tu < w.end ? w.pages[tu >> w.shift] : -1;
    r.held[u] = id >= 0 && id < w.num_pages;
    const int64_t page = r.held[u] ? id : 0;
    const uint32_t slot = (uint32_t)tu & ((1u << w.shift) - 1);
    r.key[u] = w.key + page * w.key_page + (uint64_t)slot * w.key_slot;
    r.value[u] = w.value + page * w.value_page + (uint64_t)slot * w.value_slot;
  }
  return r;
}

// Scores of a tile's tokens with the wave's queries, in units of log2 e.
template <int DT, int CT, int DP, bool FULL>
__device__ __forceinline__ void score_tile(
    const wave_state<DT, CT, DP>& st,
    const pl_u32x4 (&keys)[shape<DT, CT, DP>::kSubs][shape<DT, CT, DP>::kKeyLoads],
    int dim, float scale2, float (&p)[shape<DT, CT, DP>::kTokens]) {
  typedef shape<DT, CT, DP> S;
  pl_f32x4 s[S::kSubs];
#pragma unroll
  for (int u = 0; u < S::kSubs; ++u) {
    s[u] = pl_f32x4{0.f, 0.f, 0.f, 0.f};
    pl_f32x4 odd = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int n = 0; n < S::kKeyLoads; ++n) {
      const pl_u32x4 w = keys[u][n];
      if constexpr (CT == PL_F8E4M3) {
        const pl_u32x4 a = {widen<DT, false>(w.x), widen<DT, true>(w.x), widen<DT, false>(w.y),
                            widen<DT, true>(w.y)};
        const pl_u32x4 b = {widen<DT, false>(w.z), widen<DT, true>(w.z), widen<DT, false>(w.w),
                            widen<DT, true>(w.w)};
        s[u] = pl_mfma_chunk<DT>(a, st.query(2 * n), s[u]);
        s[u] = pl_mfma_chunk<DT>(b, st.query(2 * n + 1), s[u]);
      } else if constexpr (DT == PL_F32) {
        // two sums side by side, of the pieces that the head has
        if (FULL || n * 4 * S::E < dim) {
          if (n % 2)
            odd = pl_mfma_chunk<DT>(w, st.query(n), odd);
          else
            s[u] = pl_mfma_chunk<DT>(w, st.query(n), s[u]);
        }
      } else {
        s[u] = pl_mfma_chunk<DT>(w, st.query(n), s[u]);
      }
    }
    if constexpr (DT == PL_F32) s[u] += odd;
  }
#pragma unroll
  for (int j = 0; j < S::kTokens; ++j) p[j] = s[j / 4][j % 4] * scale2;
}

// Takes scores p and values v of a tile into the running maximum, sum and output.
template <int DT, int CT, int DP>
__device__ __forceinline__ void weigh_tile(wave_state<DT, CT, DP>& st,
                                           float (&p)[shape<DT, CT, DP>::kTokens],
                                           const uint32_t (&v)[shape<DT, CT, DP>::kTokens]
                                                              [shape<DT, CT, DP>::kVWords]) {
  typedef shape<DT, CT, DP> S;
  float top = p[0];
#pragma unroll
  for (int j = 1; j < S::kTokens; ++j) top = fmaxf(top, p[j]);
  top = fmaxf(st.m, column_max(top));
  // nothing alive yet: any finite reference gives weights of 0
  const float ref = top == -INFINITY ? 0.f : top;
  if (__any(top > st.m)) {
    const float keep = exp2_fast(st.m - ref);
    st.l *= keep;
#pragma unroll
    for (int i = 0; i < S::V; ++i) st.o[i] *= keep;
    st.m = top;
  }
#pragma unroll
  for (int j = 0; j < S::kTokens; ++j) {
    p[j] = exp2_fast(S::kLift ? p[j] - ref + S::kLift : p[j] - ref);
    st.l += p[j];
  }
  if constexpr (DT == PL_F32) {
#pragma unroll
    for (int i = 0; i < S::V; ++i) {
      pl_f32x4 part = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < S::kTokens; ++j)
        part = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v[j][i]), p[j], part, 0, 0, 0);
      st.o[i] += part;
      if (i % 2) __builtin_amdgcn_sched_barrier(0);
    }
  } else {
    pl_u32x4 part[S::kParts];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float a = p[2 * j], b = p[2 * j + 1];
#pragma unroll
      for (int k = 0; k < S::kParts; ++k) {
        // bf16's last part is exact either way
        const uint32_t x = k + 1 < S::kParts || DT == PL_BF16 ? pack2_down<DT>(a, b) : pack2<DT>(a, b);
        a -= unpack<DT>(x, 0), b -= unpack<DT>(x, 1);
        // no part negative, or 0 beside the others: an infinite value stays one
        part[k][j] = k ? at_least_smallest<DT>(x, part[0][j]) : x;
      }
    }
#pragma unroll
    for (int i = 0; i < S::V / 2; ++i) {
      uint32_t w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if constexpr (CT == PL_F8E4M3)
          w[j] = i % 2 ? widen<DT, true>(v[j][i / 2]) : widen<DT, false>(v[j][i / 2]);
        else
          w[j] = v[j][i];
      }
      pl_u32x4 a, b;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        a[j] = __builtin_amdgcn_perm(w[2 * j + 1], w[2 * j], 0x05040100);
        b[j] = __builtin_amdgcn_perm(w[2 * j + 1], w[2 * j], 0x07060302);
      }
#pragma unroll
      for (int k = 0; k < S::kParts; ++k) {
        st.o[2 * i] = pl_mfma_chunk<DT>(a, part[k], st.o[2 * i]);
        st.o[2 * i + 1] = pl_mfma_chunk<DT>(b, part[k], st.o[2 * i + 1]);
      }
      // in this order: pairing up all values first would take as many registers again
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}

// A row's tokens that count: [first, len), its atoms starting at base.
struct row_span {
  int first, len, base, atoms;
};
template <int ATOM>
__device__ __forceinline__ row_span span_of(const attend_args& a, int len) {
  const int64_t cap = a.table.num_pages ? (int64_t)a.table.max_pages << a.table.page_shift : 0;
  row_span r;
  r.len = (int)min((int64_t)max(len, 0), cap);
  r.first = a.window > 0 ? max(0, r.len - a.window) : 0;
  r.base = r.first & ~31;
  r.atoms = max(1, (r.len - r.base + ATOM - 1) / ATOM);  // an empty row's output is an atom too
  return r;
}

// Four outputs, rounded (out has the alignment of its elements alone).
template <typename T>
__device__ __forceinline__ void store4(T* p, pl_f32x4 x) {
  const T y[4] = {(T)x.x, (T)x.y, (T)x.z, (T)x.w};
  __builtin_memcpy(p, y, sizeof(y));
}
// Floats of one part: o [kCols][DP], then m and l of each column.
constexpr int part_floats(int dp) { return kCols * dp + 2 * kCols; }
template <int DP>
struct part_layout {
  static constexpr uint32_t kBytes = 4u * part_floats(DP);
  static __device__ __forceinline__ pl_buffer all(const attend_args& a) {
    return make_buffer(reinterpret_cast<uintptr_t>(a.parts), 2u * kWorkersMax * kBytes);
  }
  // Bytes of a part up to element d of column c, and up to the column's m and l.
  static __device__ __forceinline__ uint32_t at(int c, int d) { return (c * DP + d) * 4u; }
  static __device__ __forceinline__ uint32_t sums(int c) { return (kCols * DP + 2 * c) * 4u; }
};
// Parts are stored and loaded at agent scope: through to where every XCD sees
// them and from there, 16 bytes at a time.  No cache has to be invalidated for
// that (16 rows of up to 3229 tokens 18.9 -> 17.0 us, with stores of 8 bytes 17.3).
constexpr int kAgentScope = 16;

// Joins n parts (the first in slot `slot0`, part w in slot `slot` + 2 w) and
// hands each 4 finished elements of a column to `store`.  A thread takes 4
// elements over every lanes-th part, kBatch parts' loads at a time; the lanes
// join through `scratch` (6 floats a thread).
template <int DP, typename Store>
__device__ __forceinline__ void join_parts(const attend_args& a, int slot0, int slot, int n, int cols,
                                           float* scratch, Store store) {
  typedef part_layout<DP> P;
  constexpr int kBatch = 8;
  const int tid = (int)threadIdx.x, items = cols * (DP / 4);
  const int lanes = max(1, kThreads / items);
  const pl_buffer parts = P::all(a);
  for (int i0 = 0; i0 < items; i0 += kThreads) {
    const int item = i0 + (items <= kThreads ? tid % items : tid);
    const int first = items <= kThreads ? tid / items : 0;
    const bool busy = item < items && first < lanes;
    const int c = item / (DP / 4), d = item % (DP / 4) * 4;
    float m = -INFINITY, l = 0.f;
    pl_f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int w0 = first; busy && w0 < n; w0 += kBatch * lanes) {
      pl_f32x4 x[kBatch];
      float pm[kBatch], pl[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int w = min(w0 + j * lanes, n - 1);  // the last again, with no weight
        const uint32_t p = (uint32_t)(w ? slot + 2 * w : slot0) * P::kBytes;
        x[j] = __builtin_bit_cast(
            pl_f32x4, __builtin_amdgcn_raw_buffer_load_b128(parts, p + P::at(c, d), 0, kAgentScope));
        const pl_f32x2 ml = __builtin_bit_cast(
            pl_f32x2, __builtin_amdgcn_raw_buffer_load_b64(parts, p + P::sums(c), 0, kAgentScope));
        pm[j] = ml.x, pl[j] = ml.y;
      }
      float top = m;
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        pm[j] = w0 + j * lanes < n ? pm[j] : -INFINITY;
        top = fmaxf(top, pm[j]);
      }
      const float ref = top == -INFINITY ? 0.f : top, keep = exp2_fast(m - ref);
      l *= keep, o *= keep, m = top;
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const float f = exp2_fast(pm[j] - ref);
        l += f * pl[j], o += f * x[j];
      }
    }
    if (lanes > 1) {
      __syncthreads();
      if (busy) {
        float* s = scratch + 6 * tid;
        s[0] = m, s[1] = l, s[2] = o.x, s[3] = o.y, s[4] = o.z, s[5] = o.w;
      }
      __syncthreads();
      if (busy && first == 0)
        for (int k = 1; k < lanes; ++k) {
          const float* s = scratch + 6 * (k * items + item);
          const float top = fmaxf(m, s[0]), ref = top == -INFINITY ? 0.f : top;
          const float keep = exp2_fast(m - ref), f = exp2_fast(s[0] - ref);
          l = l * keep + f * s[1], m = top;
          o = o * keep + pl_f32x4{s[2], s[3], s[4], s[5]} * f;
        }
    }
    // no token gives 0; NaN, which no maximum shows, is in l and stays
    if (busy && first == 0) store(c, d, l == 0.f ? pl_f32x4{0.f, 0.f, 0.f, 0.f} : o / l);
  }
}

// How the batch's atoms are dealt out, from their number, the (row, key head)
// pairs and the longest pair.  Times are in tiles of a wave, of which a team of
// waves takes TILES for an atom: a team's first pair costs it about kFirst of
// them to begin, each pair kPair, joining parts kJoin, and waves alone read a
// batch that fills the memory kAlone times as slowly.  Measured against each other (us alone /
// team, whole / team, split): 1 row of up to 300 tokens 11.0 / 8.2 / 8.6, 64 of
// 512 19.2 / 22.5 / 26.8, 256 of 512 62 / 85 / 85, 256 of 2048 229 / 216 / 209, 1
// of 4000 88 / 39 / 11; what this takes is within a tenth of the best of them.
struct deal {
  int team;    // waves on a pair: kWaves, or 1 (no waves to join, no barrier)
  bool whole;  // pairs go whole to the run that their first atom falls in
};
constexpr float kFirst = 2.f, kPair = 8.6f, kJoin = 5.f, kAlone = 2.1f;
template <int TILES>
__device__ __forceinline__ deal choose_deal(int teams, int total, int pairs, int longest) {
  const float w = (float)teams, p = (float)pairs;
  const float n = (float)total * TILES, top = (float)longest * TILES;
  // each times w; waves enough for a pair each wait for the longest, else for a run and it
  const bool each = pairs <= (int)gridDim.x * kWaves;
  const float alone = fmaxf(kWaves * top * w + (each ? 0.f : n), kAlone * n) + w + p / kWaves;
  const float ends = kFirst * w + kPair * p;
  const float team = top * w + n + ends, split = w + n + ends + kJoin * w;
  if (alone < team && alone < split) return {1, true};
  return {kWaves, team < split};
}

template <int DT, int CT, int DP, bool FULL, bool STREAM>
__global__ __launch_bounds__(kThreads, (shape<DT, CT, DP>::kWavesPerSimd)) void pl_paged_attention_kernel(
    attend_args a) {
  typedef shape<DT, CT, DP> S;
  typedef typename pl_traits<DT>::T T;
  constexpr int kPad = 4;
  __shared__ __attribute__((aligned(16))) float s_o[kWaves][kCols][DP + kPad];
  __shared__ float s_m[kWaves][kCols], s_l[kWaves][kCols];
  __shared__ int s_last;
  const int tid = (int)threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int li = lane & 15, lg = lane >> 4;
  const int per_row = a.kv_heads * a.col_tiles;

  // Each wave works out the deal for itself: 64 rows to a look, no barrier.
  constexpr int kLooks = 4;  // that stay in registers
  int atoms[kLooks], lens[kLooks], total = 0, longest = 0;
#pragma unroll
  for (int k = 0; k < kLooks; ++k) lens[k] = a.lens[min(k * 64 + lane, a.rows - 1)];
#pragma unroll
  for (int k = 0; k < kLooks; ++k) {
    const int n = span_of<S::kAtom>(a, lens[k]).atoms;
    atoms[k] = k * 64 + lane < a.rows ? n : 0;
    total += atoms[k], longest = max(longest, atoms[k]);
  }
  for (int b = kLooks * 64 + lane; b < a.rows; b += 64) {
    const int n = span_of<S::kAtom>(a, a.lens[b]).atoms;
    total += n, longest = max(longest, n);
  }
  total = __builtin_amdgcn_readlane(scan_sum(total), 63) * per_row;
  longest = __builtin_amdgcn_readlane(scan_max(longest), 63);
  // one wave of a SIMD keeps the memory busy if its tiles are large and its products few
  const bool many =
      DT != PL_F32 && DP <= 128 && a.dim * S::kCsize >= 128 && total >= kManyAtoms;
  const int teams = many ? min((int)gridDim.x, kCus) : (int)gridDim.x;
  const deal how =
      choose_deal<S::kAtom / (kWaves * S::kTile)>(teams, total, a.rows * per_row, longest);
  const int workers = how.team == 1 ? (int)gridDim.x * kWaves : teams;
  const int worker = how.team == 1 ? wave * (int)gridDim.x + (int)blockIdx.x : (int)blockIdx.x;
  // waves enough for a pair each: no runs, whose atoms come by ones, twos and threes
  const bool each = how.team == 1 && a.rows * per_row <= workers;
  const int per = (total + workers - 1) / workers;
  const int from = (int)min((int64_t)worker * per, (int64_t)total);
  int to = min(total - per, from) + per;
  if (each ? worker >= a.rows * per_row : from >= total) return;
  // the row of its first atom: the first whose atoms up to and with it pass `from`
  int row = 0, row_start = 0, row_len = 0, at = from;
  for (int b0 = 0; !each; b0 += 64) {
    const int b = b0 + lane;
    int n = atoms[0], len = lens[0];
#pragma unroll
    for (int k = 1; k < kLooks; ++k) {
      n = b0 == k * 64 ? atoms[k] : n;
      len = b0 == k * 64 ? lens[k] : len;
    }
    if (b0 >= kLooks * 64) {
      len = b < a.rows ? a.lens[b] : 0;
      n = b < a.rows ? span_of<S::kAtom>(a, len).atoms : 0;
    }
    n *= per_row;
    const int upto = scan_sum(n) + row_start;
    const uint64_t past = __ballot(upto > from);
    if (past || b0 + 64 >= a.rows) {
      const int hit = past ? __ffsll((long long)past) - 1 : 63;
      row = b0 + hit;
      row_start = __builtin_amdgcn_readlane(upto - n, hit);
      row_len = __builtin_amdgcn_readlane(len, hit);
      break;
    }
    row_start = __builtin_amdgcn_readlane(upto, 63);
  }
  row = uniform(row);
  if (each) {
    // its pair, as if the rows before it had no atoms
    row = worker / per_row;
    row_len = as_scalar(a.lens)[row];
    row_start = 0;
    at = worker % per_row * span_of<S::kAtom>(a, row_len).atoms;
    to = at + 1;
  }
  bool skip = how.whole && !each;  // to the first pair that starts in the run
  while (at < to) {
    const row_span r = span_of<S::kAtom>(a, row_len);
    int in_row = at - row_start;
    if (skip) {
      in_row = (in_row + r.atoms - 1) / r.atoms * r.atoms;
      at = row_start + in_row;
      skip = false;
      if (at >= to) return;
    }
    if (in_row >= r.atoms * per_row) {
      row_start += r.atoms * per_row;
      row_len = as_scalar(a.lens)[++row];
      continue;
    }
    const int combo = in_row / r.atoms;
    const int pair_start = row_start + combo * r.atoms;
    const int first_atom = at - pair_start;
    const int last_atom = how.whole ? r.atoms : min(r.atoms, to - pair_start);
    const int hk = combo / a.col_tiles, ct = combo % a.col_tiles;
    const int cols = min(kCols, a.group - ct * kCols);
    const int head0 = hk * a.group + ct * kCols;

    wave_state<DT, CT, DP> st;
    st.m = -INFINITY, st.l = 0.f;
    st.q_lds = reinterpret_cast<shared_u32x4*>(&s_o[wave][0][0]) + lane;
#pragma unroll
    for (int i = 0; i < S::V; ++i) st.o[i] = pl_f32x4{0.f, 0.f, 0.f, 0.f};
    const float scale2 =
        a.scale * 1.44269504088896f * (CT == PL_F8E4M3 ? as_scalar(a.k_scale)[hk] : 1.f);

    // the tiles of this wave: every team-th of the run's
    const int end = min(r.len, r.base + last_atom * S::kAtom);
    const int step = how.team * S::kTile;
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
    // Keys of the next tile are asked for as soon as this tile's have gone into
    // the scores, values as soon as the wave is at the tile: one or the other
    // is in flight all the time, in no more registers than one tile takes.
    // Past the last tile the loads stay, of no bytes: a load that is made in
    // one turn of the loop and not in another would have to be waited for in
    // every turn.
    pl_u32x4 keys[S::kSubs][S::kKeyLoads];
    auto load_keys = [&](const tile_place<S::kSubs>& at) {
#pragma unroll
      for (int u = 0; u < S::kSubs; ++u) {
        const pl_buffer r = make_buffer(at.key[u], at.held[u] ? key_span : 0);
#pragma unroll
        for (int n = 0; n < S::kKeyLoads; ++n) {
          uint32_t x[4];
          load_words<4, STREAM>(r, key_off[n], 0, x);
          keys[u][n] = pl_u32x4{x[0], x[1], x[2], x[3]};
        }
      }
    };
    int tile = r.base + first_atom * S::kAtom + (how.team == 1 ? 0 : wave * S::kTile);
    if (tile < end) {
      tile_place<S::kSubs> place = place_tile<S::kSubs>(w, tile);
      const T* q = (const T*)a.q + row * a.q_row + (head0 + (li < cols ? li : 0)) * a.q_head;
#pragma unroll
      for (int n = 0; n < S::kSteps; ++n) {
        const int d = CT == PL_F8E4M3 ? key_piece<CT>(n / 2, lg, S::E) + (n % 2) * 8
                                      : key_piece<CT>(n, lg, S::E);
        // rows of q have the alignment of their elements alone
        pl_u32x4 x;
        __builtin_memcpy(&x, q + (FULL || d < a.dim ? d : 0), 16);
        x = li < cols && (FULL || d < a.dim) ? x : pl_u32x4{0, 0, 0, 0};
        if constexpr (S::kQueryLds)
          st.q_lds[n * 64] = x;
        else
          st.q[n] = x;
      }
      load_keys(place);
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
        float p[S::kTokens];
        score_tile<DT, CT, DP, FULL>(st, keys, a.dim, scale2, p);
        load_keys(place);
        bool whole = tile >= r.first && tile + S::kTile <= r.len;
#pragma unroll
        for (int u = 0; u < S::kSubs; ++u) whole = whole && here.held[u];
        if (!whole) {
          // slots without a token may hold anything, NaN too: no weight of 0 takes that out
#pragma unroll
          for (int j = 0; j < S::kTokens; ++j) {
            const int token = tile + 16 * (j / 4) + 4 * lg + j % 4;
            const bool alive = here.held[j / 4] && token >= r.first && token < r.len;
            p[j] = alive ? p[j] : -INFINITY;
#pragma unroll
            for (int i = 0; i < S::kVWords; ++i) v[j][i] = alive ? v[j][i] : 0u;
          }
        }
        weigh_tile<DT, CT, DP>(st, p, v);
        tile = next;
      } while (tile < end);
    }

    st.l = column_sum(st.l);
    const float v_scale = CT == PL_F8E4M3 ? as_scalar(a.v_scale)[hk] : 1.f;
    T* out = (T*)a.out + ((int64_t)row * a.heads + head0) * a.dim;
    if (how.team == 1) {
      if (li < cols) {
        const float f = st.m == -INFINITY ? 0.f : v_scale / st.l;
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int n = 0; n < S::kPieces; ++n) {
            const int d = S::value_at(4 * lg + e, n);
            T y[S::kPiece];
#pragma unroll
            for (int i = 0; i < S::kPiece; ++i) y[i] = (T)(st.o[n * S::kPiece + i][e] * f);
            // out has the alignment of its elements alone
            if (FULL || d < a.dim) __builtin_memcpy(out + li * a.dim + d, y, sizeof(y));
          }
      }
      at = pair_start + last_atom;
      continue;
    }
    // join the waves
    if (lg == 0) s_m[wave][li] = st.m, s_l[wave][li] = st.l;
    if (li < cols) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int i = 0; i < S::V; i += 4)
          *reinterpret_cast<pl_f32x4*>(
              &s_o[wave][li][S::value_at(4 * lg + e, i / S::kPiece) + i % S::kPiece]) =
              pl_f32x4{st.o[i][e], st.o[i + 1][e], st.o[i + 2][e], st.o[i + 3][e]};
    }
    __syncthreads();
    const bool complete = first_atom == 0 && last_atom == r.atoms;
    typedef part_layout<DP> P;
    const uint32_t part = (2u * blockIdx.x + (at == from ? 0 : 1)) * P::kBytes;
    const pl_buffer parts = P::all(a);
    for (int i = tid; i < cols * (DP / 4); i += kThreads) {
      const int c = i / (DP / 4), d = i % (DP / 4) * 4;
      float m = -INFINITY, l = 0.f;
      pl_f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kWaves; ++w) m = fmaxf(m, s_m[w][c]);
      const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float f = exp2_fast(s_m[w][c] - ref);
        l += f * s_l[w][c];
        o += f * *reinterpret_cast<const pl_f32x4*>(&s_o[w][c][d]);
      }
      if (complete) {
        if (FULL || d < a.dim) store4(out + c * a.dim + d, o * (m == -INFINITY ? 0.f : v_scale / l));
      } else {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(pl_u32x4, o), parts,
                                               part + P::at(c, d), 0, kAgentScope);
        if (d == 0)
          __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(pl_u32x2, pl_f32x2{m, l}), parts,
                                                part + P::sums(c), 0, kAgentScope);
      }
    }
    if (!complete) {
      // Parts are acknowledged from where every XCD sees them before the arrival
      // is counted, and the last to arrive asks for them there after that.
      const int w0 = pair_start / per, w1 = (pair_start + r.atoms - 1) / per;
      __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
      __syncthreads();
      if (tid == 0) {
        int32_t* counter = a.counters + w0 * kCounterStride;
        const int old = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        s_last = old == w1 - w0;
        if (s_last) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
      __syncthreads();
      if (s_last) {
        // the first part is its workgroup's second when that workgroup began earlier
        const int slot0 = 2 * w0 + (w0 * per == pair_start ? 0 : 1);
        join_parts<DP>(a, slot0, 2 * w0, w1 - w0 + 1, cols, &s_o[0][0][0],
                       [&](int c, int d, pl_f32x4 o) {
                         if (FULL || d < a.dim) store4(out + c * a.dim + d, o * v_scale);
                       });
      }
    }
    __syncthreads();  // the shared arrays are free again
    at = pair_start + last_atom;
  }
}

// Lines read once are marked so where a pool of pages is too large to stay in
// the GPU's last cache (256 rows of up to 1024 tokens 129 -> 120 us; 256 rows of
// up to 128, 134 MB, 20.9 -> 23.1, which a batch as small in a larger pool loses:
// how much of the pool it reads is known on the device alone).  Not where a line is read again: by the next
// 16 query heads of a key head (204 rows, 20 for each 120 -> 144 us), or,
// in heads that are no whole lines, by another load (fp32, 80 elements: 40 -> 56).
constexpr int64_t kLastCache = 256 << 20;

template <int DT, int CT, int DP>
void launch_dim(const attend_args& a, int64_t pool_bytes, dim3 grid, hipStream_t s) {
  if (a.dim != DP)
    pl_paged_attention_kernel<DT, CT, DP, false, false><<<grid, kThreads, 0, s>>>(a);
  else if (pool_bytes > kLastCache && a.col_tiles == 1)
    pl_paged_attention_kernel<DT, CT, DP, true, true><<<grid, kThreads, 0, s>>>(a);
  else
    pl_paged_attention_kernel<DT, CT, DP, true, false><<<grid, kThreads, 0, s>>>(a);
}

template <int DT, int CT>
int launch(const attend_args& a, int64_t atoms_most, hipStream_t s) {
  const int64_t pool_bytes = 2ll * a.table.num_pages * ((int64_t)a.kv_heads * a.dim << a.table.page_shift) *
                             pl_cache_elem_size(CT);
  const int64_t blocks = atoms_most < kWorkersMax ? atoms_most : kWorkersMax;
  const dim3 grid((unsigned)blocks);
  if (a.dim <= 64)
    launch_dim<DT, CT, 64>(a, pool_bytes, grid, s);
  else if (a.dim <= 128)
    launch_dim<DT, CT, 128>(a, pool_bytes, grid, s);
  else
    launch_dim<DT, CT, 256>(a, pool_bytes, grid, s);
  return pl_launch_status("pl_paged_attention");
}

}  // namespace

static_assert(PL_ATTENTION_COUNTER_INTS == kWorkersMax * kCounterStride, "one counter per workgroup");

extern "C" int64_t pl_paged_attention_workspace_bytes(int32_t dim) {
  const int dp = dim <= 64 ? 64 : dim <= 128 ? 128 : 256;
  return dim < 1 || dim > kHeadDimMax ? 0 : 2ll * kWorkersMax * part_floats(dp) * (int64_t)sizeof(float);
}

extern "C" int pl_paged_attention(int32_t dtype, int32_t cache_dtype, const void* q,
                                  const int64_t* q_strides, const void* key_cache,
                                  const int64_t* key_strides, const void* value_cache,
                                  const int64_t* value_strides, int32_t num_pages,
                                  int32_t page_size, const int32_t* page_table, int64_t table_ld,
                                  int32_t max_pages, const int32_t* lens, int32_t rows,
                                  int32_t heads, int32_t kv_heads, int32_t dim, float scale,
                                  int32_t window, const float* k_scale, const float* v_scale,
                                  void* out, void* workspace, int64_t workspace_bytes,
                                  int32_t* counters, int64_t counter_ints, void* stream) {
  const int rc = pl_check_paged("pl_paged_attention", dtype, cache_dtype, key_cache, key_strides,
                                value_cache, value_strides, num_pages, page_size, page_table,
                                table_ld, max_pages, rows, heads, kv_heads, dim, k_scale, v_scale);
  if (rc) return rc;
  if (window < 0) {
    pl_set_error("pl_paged_attention: the window is a number of tokens, or 0 for none (got %d)",
                 window);
    return PL_ERR_ARG;
  }
  if (rows == 0) return PL_OK;
  // lanes address the 16 slots of a tile with 32-bit byte offsets
  const int64_t slot_most = INT32_MAX / 16 / pl_cache_elem_size(cache_dtype);
  if (key_strides[2] < 0 || key_strides[2] > slot_most || value_strides[2] < 0 ||
      value_strides[2] > slot_most) {
    pl_set_error("pl_paged_attention: slot strides of %lld and %lld elements",
                 (long long)key_strides[2], (long long)value_strides[2]);
    return PL_ERR_LIMIT;
  }
  if (!q || !q_strides || !lens || !out) {
    pl_set_error("pl_paged_attention: null pointer");
    return PL_ERR_ARG;
  }
  const int64_t es = pl_elem_size(dtype);
  if (pl_ranges_meet(out, (int64_t)rows * heads * dim * es, q,
                     ((rows - 1) * q_strides[0] + (heads - 1) * q_strides[1] + dim) * es)) {
    pl_set_error("pl_paged_attention: out overlaps q");
    return PL_ERR_ARG;
  }
  if (!workspace || workspace_bytes < pl_paged_attention_workspace_bytes(dim) || !counters ||
      counter_ints < PL_ATTENTION_COUNTER_INTS) {
    pl_set_error("pl_paged_attention: workspace of %lld bytes and %lld counters, %lld and %d needed",
                 (long long)workspace_bytes, (long long)counter_ints,
                 (long long)pl_paged_attention_workspace_bytes(dim), PL_ATTENTION_COUNTER_INTS);
    return PL_ERR_ARG;
  }
  attend_args a;
  a.q = q, a.q_row = q_strides[0], a.q_head = q_strides[1];
  a.key = {const_cast<void*>(key_cache), key_strides[0], key_strides[1], key_strides[2]};
  a.value = {const_cast<void*>(value_cache), value_strides[0], value_strides[1], value_strides[2]};
  a.table = {page_table, table_ld, max_pages, num_pages, pl_log2_exact(page_size)};
  a.lens = lens, a.k_scale = k_scale, a.v_scale = v_scale, a.out = out, a.scale = scale;
  a.rows = rows, a.heads = heads, a.kv_heads = kv_heads, a.dim = dim, a.window = window;
  a.group = heads / kv_heads, a.col_tiles = (a.group + kCols - 1) / kCols;
  a.parts = static_cast<float*>(workspace), a.counters = counters;
  // atoms at most: every row as long as its pages or its window allow
  int64_t longest = (int64_t)max_pages * page_size;
  if (window > 0 && longest > (int64_t)window + 31) longest = (int64_t)window + 31;
  const int64_t atom = 32 * kWaves, per_pair = longest > atom ? (longest + atom - 1) / atom : 1;
  const int64_t pairs = (int64_t)rows * kv_heads * a.col_tiles;
  // token and atom numbers are 32-bit, a tile past a row's end and a run past the last one included
  if ((int64_t)max_pages * page_size > INT32_MAX - 2 * atom ||
      pairs > (INT32_MAX - kWorkersMax * kWaves) / per_pair) {
    pl_set_error("pl_paged_attention: %lld rows and key heads of up to %lld tokens are too many",
                 (long long)pairs, (long long)longest);
    return PL_ERR_LIMIT;
  }
  const int64_t atoms_most = pairs * per_pair;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (cache_dtype == PL_F8E4M3)
    return dtype == PL_BF16 ? launch<PL_BF16, PL_F8E4M3>(a, atoms_most, s)
                            : launch<PL_F16, PL_F8E4M3>(a, atoms_most, s);
  if (dtype == PL_F32) return launch<PL_F32, PL_F32>(a, atoms_most, s);
  return dtype == PL_BF16 ? launch<PL_BF16, PL_BF16>(a, atoms_most, s)
                          : launch<PL_F16, PL_F16>(a, atoms_most, s);
}
