// What the two attentions over a paged cache share: tiles of tokens from their pages
// to registers, 16 query columns to a matrix product, parts of a row and their join.
#pragma once

#include "pl_paged.h"

namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr int kCols = 16;  // query heads of a workgroup's products
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

// Four outputs, rounded (out has the alignment of its elements alone).
template <typename T>
__device__ __forceinline__ void store4(T* p, pl_f32x4 x) {
  const T y[4] = {(T)x.x, (T)x.y, (T)x.z, (T)x.w};
  __builtin_memcpy(p, y, sizeof(y));
}
constexpr int kLine = 128;  // bytes of an L2's line, which a workspace begins with
inline bool on_a_line(const void* p) { return reinterpret_cast<uintptr_t>(p) % kLine == 0; }
// Floats of one part: o [kCols][DP], then m and l of each column.
constexpr int part_floats(int dp) { return kCols * dp + 2 * kCols; }
template <int DP>
struct part_layout {
  static constexpr uint32_t kBytes = 4u * part_floats(DP);
  static_assert(kBytes % kLine == 0, "no line holds two workgroups' parts (arrive_last)");
  static __device__ __forceinline__ pl_buffer all(const float* parts, uint32_t n) {
    return make_buffer(reinterpret_cast<uintptr_t>(parts), n * kBytes);
  }
  // Bytes of a part up to element d of column c, and up to the column's m and l.
  static __device__ __forceinline__ uint32_t at(int c, int d) { return (c * DP + d) * 4u; }
  static __device__ __forceinline__ uint32_t sums(int c) { return (kCols * DP + 2 * c) * 4u; }
};
// Parts are stored and loaded at agent scope: through to where every XCD sees
// them and from there, 16 bytes at a time.  No cache has to be invalidated for
// that (16 rows of up to 3229 tokens 18.9 -> 17.0 us, with stores of 8 bytes 17.3).
constexpr int kAgentScope = 16;

// Arrival of a workgroup whose parts of a pair are stored: whether it is the last of `others` + 1,
// which then may read what the others have stored.  Every thread calls it; the counter is 0 again
// behind the last.
//
// The order is the hardware's: a wave's stores at agent scope go through its XCD's L2 to memory, and
// vmcnt counts them until they are there; every wave has waited for its own, and the barrier
// for the others', before the arrival is counted, and the last one asks for the parts after its
// own count has come back.  No L2 answers it from an older copy: a part is whole 128-byte lines of one workgroup, nobody asks
// for them before all have arrived, and a launch begins with the L2s invalidated.  (Records that share lines
// between workgroups have no such promise.)  A release and an acquire at the counter instead write
// back and invalidate a whole L2 at every arrival: 64 rows of 8 drafts over 4096 tokens 156 -> 178 us, 64
// rows over 8192 tokens in 8 bits 108 -> 131.
__device__ __forceinline__ bool arrive_last(int32_t* counter, int others, int* s_last) {
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  __syncthreads();
  if (threadIdx.x == 0) {
    const int old = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *s_last = old == others;
    if (old == others) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  return *s_last != 0;
}

// Joins n parts (the first in slot `slot0`, part w in slot `slot` + `step` w) and
// hands each 4 finished elements of a column to `store`.  A thread takes 4
// elements over every lanes-th part, kBatch parts' loads at a time; the lanes
// join through `scratch` (6 floats a thread).
template <int DP, typename Store>
__device__ __forceinline__ void join_parts(pl_buffer parts, int slot0, int slot, int step, int n, int cols,
                                           float* scratch, Store store) {
  typedef part_layout<DP> P;
  constexpr int kBatch = 8;
  const int tid = (int)threadIdx.x, items = cols * (DP / 4);
  const int lanes = max(1, kThreads / items);
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
        const uint32_t p = (uint32_t)(w ? slot + step * w : slot0) * P::kBytes;
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

}  // namespace
