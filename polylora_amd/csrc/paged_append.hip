// Rotation by position and append to a paged key-value cache, with the norms of
// queries and keys in the same pass where a model has them.
#include <algorithm>

#include "pl_paged.h"

int pl_check_paged(const char* what, int32_t dtype, int32_t cache_dtype, const void* key_cache,
                   const int64_t* key_strides, const void* value_cache,
                   const int64_t* value_strides, int32_t num_pages, int32_t page_size,
                   const int32_t* page_table, int64_t table_ld, int32_t max_pages, int32_t rows,
                   int32_t heads, int32_t kv_heads, int32_t dim, const float* k_scale,
                   const float* v_scale) {
  if (dtype != PL_F32 && dtype != PL_BF16 && dtype != PL_F16) {
    pl_set_error("%s: unknown element type %d", what, dtype);
    return PL_ERR_ARG;
  }
  const bool fp8 = cache_dtype == PL_F8E4M3;
  if (cache_dtype != dtype && !(fp8 && dtype != PL_F32)) {
    pl_set_error("%s: the cache holds the model's element type, or e4m3 for 16-bit models", what);
    return PL_ERR_ARG;
  }
  if (fp8 != (k_scale != nullptr) || fp8 != (v_scale != nullptr)) {
    pl_set_error("%s: scales belong to an e4m3 cache, one for each key head", what);
    return PL_ERR_ARG;
  }
  if (rows < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads != 0) {
    pl_set_error("%s: bad sizes (rows %d, heads %d, key heads %d)", what, rows, heads, kv_heads);
    return PL_ERR_ARG;
  }
  if (dim < kHeadDimStep || dim > kHeadDimMax || dim % kHeadDimStep != 0) {
    pl_set_error("%s: the head size is a multiple of %d up to %d (got %d)", what, kHeadDimStep,
                 kHeadDimMax, dim);
    return PL_ERR_LIMIT;
  }
  if (page_size < kPageMin || page_size > kPageMax || pl_log2_exact(page_size) < 0) {
    pl_set_error("%s: a page holds a power of two of at least %d tokens (got %d)", what, kPageMin,
                 page_size);
    return PL_ERR_LIMIT;
  }
  if (num_pages < 0 || max_pages < 0 || (table_ld < max_pages && table_ld != 0) ||
      (int64_t)max_pages * page_size > INT32_MAX) {
    pl_set_error("%s: bad page table (pages %d, columns %d, row stride %lld)", what, num_pages,
                 max_pages, (long long)table_ld);
    return PL_ERR_ARG;
  }
  if (rows > 0 && ((!page_table && max_pages > 0) || !key_strides || !value_strides ||
                   (num_pages > 0 && (!key_cache || !value_cache)))) {
    pl_set_error("%s: null pointer", what);
    return PL_ERR_ARG;
  }
  if (rows > 0) {
    // rows of a head are read and written in 16-byte pieces
    const int64_t e = 16 / pl_cache_elem_size(cache_dtype);
    bool ok = reinterpret_cast<uintptr_t>(key_cache) % 16 == 0 &&
              reinterpret_cast<uintptr_t>(value_cache) % 16 == 0;
    const int32_t sizes[3] = {num_pages, kv_heads, page_size};
    for (int i = 0; i < 3; ++i)  // a dimension of one is never stepped along
      ok = ok && (sizes[i] <= 1 || (key_strides[i] % e == 0 && value_strides[i] % e == 0));
    if (!ok) {
      pl_set_error("%s: cache pointers and strides must be whole 16-byte pieces", what);
      return PL_ERR_ALIGN;
    }
  }
  return PL_OK;
}

bool pl_elements_apart(const int64_t* strides, int32_t pages, int32_t kv_heads, int32_t page_size,
                       int32_t dim) {
  struct {
    int64_t stride, size;
  } d[3] = {{strides[0], pages}, {strides[1], kv_heads}, {strides[2], page_size}};
  std::sort(d, d + 3, [](const auto& x, const auto& y) { return x.stride < y.stride; });
  int64_t reach = dim;
  for (const auto& x : d) {
    if (x.size == 1) continue;
    if (x.stride < reach) return false;
    reach += (x.size - 1) * x.stride;
  }
  return true;
}

namespace {

constexpr int kThreads = 256;
// Workgroups that fill the GPU (eight on each of 256 CUs).
constexpr int kFullGrid = 2048;
// Workgroups up to which a token's heads are shared out.
constexpr int kFewTokens = 512;
// Outputs above this pass by the caches, where the next launch, on other XCDs,
// would hardly find them (32 x 1024 prompt tokens 135 -> 127 us, 8 x 64 5.6 ->
// 4.9; 256 single tokens are not worth it, 4.8 -> 5.0).
constexpr int64_t kCacheBytes = 4 << 20;

struct append_args {
  const void *q, *k, *v;
  int64_t qs[3], ks[3], vs[3];  // row, token, head strides
  void *q_out, *k_out;          // contiguous [rows][row_len][heads][dim]; k_out may be null
  pl_cache_view key, value;
  pl_page_table table;
  const int32_t *past, *seq_lens;
  const float *cos, *sin;  // [positions][rot / 2]
  const float *k_scale, *v_scale;
  int32_t rows, row_len, heads, kv_heads, dim, positions, half, interleaved;
  int32_t turns, units, group;  // places of a head that turn, all of them, tokens of a workgroup
};

// The scale of an e4m3 cache's head and its reciprocal.
struct e4m3_scale {
  float s, per;
};
template <int CT>
__device__ __forceinline__ e4m3_scale head_scale(const float* scales, int head) {
  const float s = CT == PL_F8E4M3 ? scales[head] : 1.f;
  return {s, 1.f / s};
}
// A value over the scale, saturated (NaN stays NaN).  The product with the
// scale's reciprocal, taken once for a head, is off by its roundings, which show
// half way between two e4m3 numbers; what it leaves of x corrects it, where it
// is not saturated anyway (dividing each value: 24 x 77 tokens 7.3 -> 8.1 us).
__device__ __forceinline__ float to_e4m3_range(float x, e4m3_scale scale) {
  const float z = x * scale.per;
  const float y = fabsf(z) < 2 * kE4M3Max ? fmaf(fmaf(-z, scale.s, x), scale.per, z) : z;
  return y != y ? y : fminf(fmaxf(y, -kE4M3Max), kE4M3Max);
}

// VEC elements of a row as fp32, and their stores.
template <int DT, int VEC>
__device__ __forceinline__ void load_vec(const void* p, int64_t at, float (&x)[VEC]) {
  typedef typename pl_traits<DT>::T T;
  typedef T TV __attribute__((ext_vector_type(VEC)));
  const T* q = (const T*)p + at;
  if constexpr (VEC == 1) {
    x[0] = (float)*q;
  } else {
    const TV v = *reinterpret_cast<const TV*>(q);
#pragma unroll
    for (int e = 0; e < VEC; ++e) x[e] = (float)v[e];
  }
}
// STREAM: past the caches, for outputs larger than they are.
template <int DT, int VEC, bool STREAM>
__device__ __forceinline__ void store_vec(void* p, int64_t at, const float (&x)[VEC]) {
  typedef typename pl_traits<DT>::T T;
  typedef T TV __attribute__((ext_vector_type(VEC)));
  T* q = (T*)p + at;
  if constexpr (VEC == 1) {
    *q = (T)x[0];
  } else {
    TV v;
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = (T)x[e];
    if constexpr (STREAM)
      __builtin_nontemporal_store(v, reinterpret_cast<TV*>(q));
    else
      *reinterpret_cast<TV*>(q) = v;
  }
}
template <int DT, int CT, int VEC, bool STREAM>
__device__ __forceinline__ void store_cache(void* p, int64_t at, const float (&x)[VEC], e4m3_scale scale) {
  if constexpr (CT == PL_F8E4M3) {
    uint8_t* q = (uint8_t*)p + at;
    uint32_t w[(VEC + 3) / 4] = {};
#pragma unroll
    for (int e = 0; e < VEC; e += 2) {
      const float lo = to_e4m3_range(x[e], scale);
      const float hi = e + 1 < VEC ? to_e4m3_range(x[e + 1], scale) : lo;
      w[e / 4] = e % 4 ? __builtin_amdgcn_cvt_pk_fp8_f32(lo, hi, (int)w[e / 4], true)
                       : __builtin_amdgcn_cvt_pk_fp8_f32(lo, hi, (int)w[e / 4], false);
    }
    __builtin_memcpy(__builtin_assume_aligned(q, VEC), w, VEC);
  } else {
    store_vec<DT, VEC, STREAM>(p, at, x);
  }
}

// A workgroup takes `group` tokens (or one of gridDim.y shares of them).  A
// thread keeps one place of the head, VEC elements and, split in halves, the
// VEC that turn against them, and walks the token's query and key heads with it,
// so that it reads its part of cos and sin once; the threads then copy the values.
//
// Bound by memory: every element of q, k and v is read and written once.  Few
// tokens are bound by reads that wait for each other: length, position, page
// and angles, then of a head its first half and its second, an 8-bit cache's
// scale, and after the heads the values (256 single tokens 4.4 us, 1.2 of it bytes).
template <int DT, int CT, int VEC, bool STREAM>
__global__ __launch_bounds__(kThreads) void pl_rope_append_kernel(append_args a) {
  const int tid = (int)threadIdx.x;
  // threads of a token, and this thread's
  const int part = kThreads / a.group;
  const int sub = tid / part, rank = tid - sub * part;
  const int64_t token = (int64_t)blockIdx.x * a.group + sub;
  if (token >= (int64_t)a.rows * a.row_len) return;
  const int b = (int)(token / a.row_len), t = (int)(token - (int64_t)b * a.row_len);
  const int n = a.seq_lens ? min(a.seq_lens[b], a.row_len) : a.row_len;
  const int64_t pos = (int64_t)a.past[b] + t, column = pos >> a.table.page_shift;
  int page = -1;
  if (t < n && pos >= 0 && pos < a.positions && column < a.table.max_pages)
    page = a.table.p[b * a.table.ld + column];
  const bool live = page >= 0 && page < a.table.num_pages;
  const int64_t slot = pos & ((1 << a.table.page_shift) - 1);

  // query and key heads: place u of the head for heads lane, lane + lanes, ...
  const int lanes = part / a.units, lane = rank / a.units, u = rank - lane * a.units;
  if (lane < lanes) {
    // the first `turns` places turn, each against the place half a rotation on
    // or, interleaved, in pairs inside (a place of one element against the
    // next); the rest are copied
    const bool turn = u < a.turns, split = turn && (VEC == 1 || !a.interleaved);
    const int d = !turn                           ? 2 * a.half + (u - a.turns) * VEC
                  : VEC == 1 && a.interleaved ? 2 * u
                                                  : u * VEC;
    const int d2 = !split ? d : a.interleaved ? d + 1 : d + a.half;
    float c[VEC], s[VEC];  // interleaved: VEC / 2 of them
    if (turn && live) {
      const int64_t i = pos * a.half + (a.interleaved ? d >> 1 : d);
      if (VEC > 1 && a.interleaved) {
        __builtin_memcpy(c, a.cos + i, VEC / 2 * sizeof(float));
        __builtin_memcpy(s, a.sin + i, VEC / 2 * sizeof(float));
      } else {
        __builtin_memcpy(c, a.cos + i, VEC * sizeof(float));
        __builtin_memcpy(s, a.sin + i, VEC * sizeof(float));
      }
    }
    const int step = lanes * (int)gridDim.y;
    for (int h = (int)blockIdx.y * lanes + lane; h < a.heads + a.kv_heads; h += step) {
      const bool is_q = h < a.heads;
      const int hh = is_q ? h : h - a.heads;
      float x[VEC], y[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) x[e] = y[e] = 0.f;
      if (live) {
        const void* src = is_q ? a.q : a.k;
        const int64_t at = is_q ? b * a.qs[0] + t * a.qs[1] + hh * a.qs[2]
                                : b * a.ks[0] + t * a.ks[1] + hh * a.ks[2];
        load_vec<DT, VEC>(src, at + d, x);
        if (split) load_vec<DT, VEC>(src, at + d2, y);
        if (split) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float x0 = x[e], y0 = y[e];
            x[e] = x0 * c[e] - y0 * s[e];
            y[e] = y0 * c[e] + x0 * s[e];
          }
        } else if (turn) {
#pragma unroll
          for (int e = 0; e + 1 < VEC; e += 2) {
            const float x0 = x[e], y0 = x[e + 1];
            x[e] = x0 * c[e / 2] - y0 * s[e / 2];
            x[e + 1] = y0 * c[e / 2] + x0 * s[e / 2];
          }
        }
      }
      void* dense = is_q ? a.q_out : a.k_out;
      if (dense) {
        const int64_t at = (token * (is_q ? a.heads : a.kv_heads) + hh) * a.dim;
        store_vec<DT, VEC, STREAM>(dense, at + d, x);
        if (split) store_vec<DT, VEC, STREAM>(dense, at + d2, y);
      }
      if (!is_q && live) {
        const int64_t at = page * a.key.s_page + hh * a.key.s_head + slot * a.key.s_slot;
        const e4m3_scale scale = head_scale<CT>(a.k_scale, hh);
        store_cache<DT, CT, VEC, STREAM>(a.key.p, at + d, x, scale);
        if (split) store_cache<DT, CT, VEC, STREAM>(a.key.p, at + d2, y, scale);
      }
    }
  }
  if (!live) return;
  const int places = a.dim / VEC;
  for (int i = (int)blockIdx.y * part + rank; i < a.kv_heads * places; i += part * (int)gridDim.y) {
    const int hh = i / places, d = (i - hh * places) * VEC;
    float x[VEC];
    load_vec<DT, VEC>(a.v, b * a.vs[0] + t * a.vs[1] + hh * a.vs[2] + d, x);
    store_cache<DT, CT, VEC, STREAM>(a.value.p,
                                     page * a.value.s_page + hh * a.value.s_head + slot * a.value.s_slot + d,
                                     x, head_scale<CT>(a.v_scale, hh));
  }
}

// With the norms of queries and keys of each head in the same pass,
//   x / sqrt(mean(x^2) + eps) * w, then the rotation, fp32, rounded once,
// and with a token's depth in a tree of drafts as its distance from the row's
// last token (its slot stays past + t).
struct norm_args {
  const void *q_w, *k_w;  // [dim], null for no norm
  int32_t wide;           // weights are fp32, else the model's type
  float eps;
  const int32_t* depths;  // [rows][depths_ld], null for t
  int64_t depths_ld;
  int32_t lanes;          // of a head: a power of two up to 64
};

// Sum over the lanes of a head: aligned groups of `lanes`, the result in each.
// Inside 16 lanes by row moves (pairs, pairs of pairs, halves and whole rows
// mirrored), beyond them by the row swaps.
template <int CTRL>
__device__ __forceinline__ float plus_moved(float x) {
  return x + __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ float head_sum(float x, int lanes) {
  if (lanes > 1) x = plus_moved<0xb1>(x);   // lane ^ 1
  if (lanes > 2) x = plus_moved<0x4e>(x);   // lane ^ 2
  if (lanes > 4) x = plus_moved<0x141>(x);  // 7 - lane
  if (lanes > 8) x = plus_moved<0x140>(x);  // 15 - lane
  if (lanes > 16) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if (lanes > 32) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return x;
}

// The kernel above with a head on `lanes` lanes side by side, PER places of the
// head to a lane (more than one only where places are too small for 64 lanes to
// hold a head), so that its sum of squares stays inside a wave: x / sqrt(mean x^2 + eps) times
// the head's weights, in fp32, then the rotation, with no rounding between.  Memory bounds
// it: prompts of 32 x 1024 tokens (32 + 8 + 8 heads of 128, bf16) take 132 us, 5.1 TB/s, a copy's
// rate; one row of 6 tokens 5.6 us, a chain of reads.
template <int DT, int CT, int VEC, bool STREAM>
__global__ __launch_bounds__(kThreads) void pl_norm_rope_append_kernel(append_args a, norm_args n) {
  constexpr int PER = VEC >= 4 ? 1 : 4 / VEC;
  const int tid = (int)threadIdx.x;
  const int part = kThreads / a.group;  // whole waves
  const int sub = tid / part, rank = tid - sub * part;
  const int64_t token = (int64_t)blockIdx.x * a.group + sub;
  if (token >= (int64_t)a.rows * a.row_len) return;
  const int b = (int)(token / a.row_len), t = (int)(token - (int64_t)b * a.row_len);
  const int count = a.seq_lens ? min(a.seq_lens[b], a.row_len) : a.row_len;
  const int64_t past = a.past[b], at_slot = past + t, column = at_slot >> a.table.page_shift;
  const int64_t pos = past + (n.depths ? n.depths[b * n.depths_ld + t] : t);
  int page = -1;
  if (t < count && at_slot >= 0 && pos >= 0 && pos < a.positions && column < a.table.max_pages)
    page = a.table.p[b * a.table.ld + column];
  const bool live = page >= 0 && page < a.table.num_pages;
  const int64_t slot = at_slot & ((1 << a.table.page_shift) - 1);

  const int heads_at_once = part / n.lanes, lane = rank / n.lanes, u0 = rank - lane * n.lanes;
  bool has[PER], turn[PER], split[PER];
  int d[PER], d2[PER];
  float c[PER][VEC], s[PER][VEC], wq[PER][2][VEC], wk[PER][2][VEC];
  auto load_weight = [&](const void* w, int at, float (&x)[VEC]) {
    if (n.wide)
      load_vec<PL_F32, VEC>(w, at, x);
    else
      load_vec<DT, VEC>(w, at, x);
  };
#pragma unroll
  for (int p = 0; p < PER; ++p) {
    const int u = u0 + p * n.lanes;
    has[p] = live && u < a.units;
    turn[p] = u < a.turns, split[p] = turn[p] && (VEC == 1 || !a.interleaved);
    d[p] = !turn[p]                   ? 2 * a.half + (u - a.turns) * VEC
           : VEC == 1 && a.interleaved ? 2 * u
                                       : u * VEC;
    d2[p] = !split[p] ? d[p] : a.interleaved ? d[p] + 1 : d[p] + a.half;
    if (!has[p]) continue;
    if (turn[p]) {
      const int64_t i = pos * a.half + (a.interleaved ? d[p] >> 1 : d[p]);
      if (VEC > 1 && a.interleaved) {
        __builtin_memcpy(c[p], a.cos + i, VEC / 2 * sizeof(float));
        __builtin_memcpy(s[p], a.sin + i, VEC / 2 * sizeof(float));
      } else {
        __builtin_memcpy(c[p], a.cos + i, VEC * sizeof(float));
        __builtin_memcpy(s[p], a.sin + i, VEC * sizeof(float));
      }
    }
    if (n.q_w) load_weight(n.q_w, d[p], wq[p][0]), load_weight(n.q_w, d2[p], wq[p][1]);
    if (n.k_w) load_weight(n.k_w, d[p], wk[p][0]), load_weight(n.k_w, d2[p], wk[p][1]);
  }
  const int step = heads_at_once * (int)gridDim.y;
  // the same turns for every lane: a head's lanes sum up together
  for (int h0 = (int)blockIdx.y * heads_at_once; h0 < a.heads + a.kv_heads; h0 += step) {
    const int h = h0 + lane;
    const bool head = lane < heads_at_once && h < a.heads + a.kv_heads;
    const bool is_q = h < a.heads;
    const int hh = is_q ? h : h - a.heads;
    float x[PER][VEC], y[PER][VEC], squares = 0.f;
#pragma unroll
    for (int p = 0; p < PER; ++p) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) x[p][e] = y[p][e] = 0.f;
      if (head && has[p]) {
        const void* src = is_q ? a.q : a.k;
        const int64_t at = is_q ? b * a.qs[0] + t * a.qs[1] + hh * a.qs[2]
                                : b * a.ks[0] + t * a.ks[1] + hh * a.ks[2];
        load_vec<DT, VEC>(src, at + d[p], x[p]);
        if (split[p]) load_vec<DT, VEC>(src, at + d2[p], y[p]);
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) squares += x[p][e] * x[p][e] + y[p][e] * y[p][e];
    }
    const float r = 1.f / sqrtf(head_sum(squares, n.lanes) / (float)a.dim + n.eps);
    if (!head) continue;
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      if (u0 + p * n.lanes >= a.units) continue;
      if (live) {
        if (is_q ? n.q_w != nullptr : n.k_w != nullptr) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            x[p][e] = x[p][e] * r * (is_q ? wq[p][0][e] : wk[p][0][e]);
            if (split[p]) y[p][e] = y[p][e] * r * (is_q ? wq[p][1][e] : wk[p][1][e]);
          }
        }
        if (split[p]) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float x0 = x[p][e], y0 = y[p][e];
            x[p][e] = x0 * c[p][e] - y0 * s[p][e];
            y[p][e] = y0 * c[p][e] + x0 * s[p][e];
          }
        } else if (turn[p]) {
#pragma unroll
          for (int e = 0; e + 1 < VEC; e += 2) {
            const float x0 = x[p][e], y0 = x[p][e + 1];
            x[p][e] = x0 * c[p][e / 2] - y0 * s[p][e / 2];
            x[p][e + 1] = y0 * c[p][e / 2] + x0 * s[p][e / 2];
          }
        }
      }
      void* dense = is_q ? a.q_out : a.k_out;
      if (dense) {
        const int64_t at = (token * (is_q ? a.heads : a.kv_heads) + hh) * a.dim;
        store_vec<DT, VEC, STREAM>(dense, at + d[p], x[p]);
        if (split[p]) store_vec<DT, VEC, STREAM>(dense, at + d2[p], y[p]);
      }
      if (!is_q && live) {
        const int64_t at = page * a.key.s_page + hh * a.key.s_head + slot * a.key.s_slot;
        const e4m3_scale scale = head_scale<CT>(a.k_scale, hh);
        store_cache<DT, CT, VEC, STREAM>(a.key.p, at + d[p], x[p], scale);
        if (split[p]) store_cache<DT, CT, VEC, STREAM>(a.key.p, at + d2[p], y[p], scale);
      }
    }
  }
  if (!live) return;
  const int places = a.dim / VEC;
  for (int i = (int)blockIdx.y * part + rank; i < a.kv_heads * places; i += part * (int)gridDim.y) {
    const int hh = i / places, at = (i - hh * places) * VEC;
    float x[VEC];
    load_vec<DT, VEC>(a.v, b * a.vs[0] + t * a.vs[1] + hh * a.vs[2] + at, x);
    store_cache<DT, CT, VEC, STREAM>(a.value.p,
                                     page * a.value.s_page + hh * a.value.s_head + slot * a.value.s_slot + at,
                                     x, head_scale<CT>(a.v_scale, hh));
  }
}

// One of the two kernels; `n` null for the first.
template <int DT, int CT, int VEC, bool STREAM>
void launch_one(const append_args& a, const norm_args* n, dim3 grid, hipStream_t s) {
  if (n)
    pl_norm_rope_append_kernel<DT, CT, VEC, STREAM><<<grid, kThreads, 0, s>>>(a, *n);
  else
    pl_rope_append_kernel<DT, CT, VEC, STREAM><<<grid, kThreads, 0, s>>>(a);
}

template <int DT, int CT, bool STREAM>
void launch_vec(const append_args& a, const norm_args* n, int vec, dim3 grid, hipStream_t s) {
  if (vec == 8) {
    if constexpr (DT != PL_F32) launch_one<DT, CT, 8, STREAM>(a, n, grid, s);
  } else if (vec == 4) {
    launch_one<DT, CT, 4, STREAM>(a, n, grid, s);
  } else if (vec == 2) {
    launch_one<DT, CT, 2, STREAM>(a, n, grid, s);
  } else {
    launch_one<DT, CT, 1, STREAM>(a, n, grid, s);
  }
}

template <int DT, int CT>
int launch(const char* what, append_args a, norm_args* n, int vec, hipStream_t s) {
  // places of a head that a thread may keep
  a.turns = (a.interleaved && vec > 1 ? 2 * a.half : a.half) / vec;
  a.units = a.turns + (a.dim - 2 * a.half) / vec;
  int threads = a.units;  // of a head
  if (n) {
    n->lanes = 1;
    while (n->lanes < a.units && n->lanes < 64) n->lanes *= 2;
    threads = n->lanes;
  }
  const int64_t tokens = (int64_t)a.rows * a.row_len;
  // one token per workgroup while that leaves some idle, then enough of them
  // that every thread walks several heads with the angles it has read
  a.group = 1;
  while (a.group < 4 && tokens / (2 * a.group) >= kFullGrid && kThreads / (2 * a.group) >= threads)
    a.group *= 2;
  // few tokens: as many workgroups to each as have a head for every thread
  // (2 tokens of 64 + 8 heads of 256: 8.5 -> 4.1 us)
  int shares = 1;
  while (tokens * shares < kFewTokens && (a.heads + a.kv_heads) * threads > kThreads * shares) shares *= 2;
  const dim3 grid((unsigned)((tokens + a.group - 1) / a.group), (unsigned)shares);
  const int64_t bytes = tokens * (a.heads + 2 * a.kv_heads) * a.dim * pl_elem_size(DT);
  if (bytes > kCacheBytes)
    launch_vec<DT, CT, true>(a, n, vec, grid, s);
  else
    launch_vec<DT, CT, false>(a, n, vec, grid, s);
  return pl_launch_status(what);
}

// Both entry points; `n` null for the one without norms and depths.
int append(const char* what, int32_t dtype, int32_t cache_dtype, const void* q,
           const int64_t* q_strides, const void* k, const int64_t* k_strides,
           const void* v, const int64_t* v_strides, void* q_out, void* k_out,
           void* key_cache, const int64_t* key_strides, void* value_cache,
           const int64_t* value_strides, int32_t num_pages, int32_t page_size,
           const int32_t* page_table, int64_t table_ld, int32_t max_pages,
           const int32_t* past_lens, const int32_t* seq_lens, int32_t rows,
           int32_t row_len, int32_t heads, int32_t kv_heads, int32_t dim,
           const float* cos, const float* sin, int32_t positions, int32_t rot,
           int32_t interleaved, const float* k_scale, const float* v_scale,
           norm_args* n, void* stream) {
  const int rc = pl_check_paged(what, dtype, cache_dtype, key_cache, key_strides,
                                value_cache, value_strides, num_pages, page_size, page_table,
                                table_ld, max_pages, rows, heads, kv_heads, dim, k_scale, v_scale);
  if (rc) return rc;
  if (row_len < 0 || rot < 0 || rot > dim || rot % 2 != 0 || positions < 0) {
    pl_set_error("%s: bad sizes (row_len %d, rot %d of %d, positions %d)", what, row_len, rot, dim,
                 positions);
    return PL_ERR_ARG;
  }
  const int64_t tokens = (int64_t)rows * row_len;
  if (tokens == 0) return PL_OK;
  if (!q || !k || !v || !q_out || !q_strides || !k_strides || !v_strides || !past_lens ||
      (rot > 0 && positions > 0 && (!cos || !sin))) {
    pl_set_error("%s: null pointer", what);
    return PL_ERR_ARG;
  }
  const int64_t es = pl_elem_size(dtype), q_bytes = tokens * heads * dim * es;
  const int64_t k_bytes = tokens * kv_heads * dim * es;
  auto reach = [&](const int64_t* s, int n) {
    return ((rows - 1) * s[0] + (row_len - 1) * s[1] + (n - 1) * s[2] + dim) * es;
  };
  const void* inputs[3] = {q, k, v};
  const int64_t reaches[3] = {reach(q_strides, heads), reach(k_strides, kv_heads),
                              reach(v_strides, kv_heads)};
  for (int i = 0; i < 3; ++i)
    if (pl_ranges_meet(q_out, q_bytes, inputs[i], reaches[i]) ||
        pl_ranges_meet(k_out, k_out ? k_bytes : 0, inputs[i], reaches[i])) {
      pl_set_error("%s: an output overlaps an input", what);
      return PL_ERR_ARG;
    }
  if (!pl_grid_fits(tokens, kThreads)) {
    pl_set_error("%s: too many tokens (%lld)", what, (long long)tokens);
    return PL_ERR_LIMIT;
  }
  if (num_pages > 0 && (key_cache == value_cache ||
                        !pl_elements_apart(key_strides, num_pages, kv_heads, page_size, dim) ||
                        !pl_elements_apart(value_strides, num_pages, kv_heads, page_size, dim))) {
    pl_set_error("%s: elements of the caches share their places", what);
    return PL_ERR_ARG;
  }
  append_args a;
  a.q = q, a.k = k, a.v = v;
  for (int i = 0; i < 3; ++i) a.qs[i] = q_strides[i], a.ks[i] = k_strides[i], a.vs[i] = v_strides[i];
  a.q_out = q_out, a.k_out = k_out;
  a.key = {key_cache, key_strides[0], key_strides[1], key_strides[2]};
  a.value = {value_cache, value_strides[0], value_strides[1], value_strides[2]};
  a.table = {page_table, table_ld, max_pages, num_pages, pl_log2_exact(page_size)};
  a.past = past_lens, a.seq_lens = seq_lens, a.cos = cos, a.sin = sin;
  a.k_scale = k_scale, a.v_scale = v_scale;
  a.rows = rows, a.row_len = row_len, a.heads = heads, a.kv_heads = kv_heads, a.dim = dim;
  a.positions = positions, a.half = rot / 2, a.interleaved = interleaved;
  // Elements a thread moves at once: 16 bytes' worth where the halves of a
  // rotation, and every pointer and stride, are whole pieces of that many.
  auto whole = [&](int vec) {
    const uintptr_t bytes = (uintptr_t)vec * es;
    bool ok = (a.interleaved ? rot : rot / 2) % vec == 0 && dim % vec == 0;
    const void* pointers[5] = {q, k, v, q_out, k_out};
    for (const void* p : pointers) ok = ok && reinterpret_cast<uintptr_t>(p) % bytes == 0;
    for (int i = 0; i < 3; ++i)
      ok = ok && a.qs[i] % vec == 0 && a.ks[i] % vec == 0 && a.vs[i] % vec == 0;
    if (n)
      for (const void* w : {n->q_w, n->k_w})
        ok = ok && reinterpret_cast<uintptr_t>(w) % (vec * (n->wide ? 4 : es)) == 0;
    return ok;
  };
  int vec = (int)(16 / es);
  while (vec > 1 && !whole(vec)) vec /= 2;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (cache_dtype == PL_F8E4M3)
    return dtype == PL_BF16 ? launch<PL_BF16, PL_F8E4M3>(what, a, n, vec, s)
                            : launch<PL_F16, PL_F8E4M3>(what, a, n, vec, s);
  if (dtype == PL_F32) return launch<PL_F32, PL_F32>(what, a, n, vec, s);
  return dtype == PL_BF16 ? launch<PL_BF16, PL_BF16>(what, a, n, vec, s)
                          : launch<PL_F16, PL_F16>(what, a, n, vec, s);
}

}  // namespace

extern "C" int pl_rope_append(int32_t dtype, int32_t cache_dtype, const void* q, const int64_t* q_strides,
    const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides, void* q_out,
    void* k_out, void* key_cache, const int64_t* key_strides, void* value_cache,
    const int64_t* value_strides, int32_t num_pages, int32_t page_size, const int32_t* page_table,
    int64_t table_ld, int32_t max_pages, const int32_t* past_lens, const int32_t* seq_lens, int32_t rows,
    int32_t row_len, int32_t heads, int32_t kv_heads, int32_t dim, const float* cos, const float* sin,
    int32_t positions, int32_t rot, int32_t interleaved, const float* k_scale, const float* v_scale,
    void* stream) {
  return append("pl_rope_append", dtype, cache_dtype, q, q_strides, k, k_strides, v, v_strides, q_out, k_out, key_cache, key_strides,
                value_cache, value_strides, num_pages, page_size, page_table, table_ld, max_pages, past_lens, seq_lens,
                rows, row_len, heads, kv_heads, dim, cos, sin, positions, rot, interleaved, k_scale, v_scale, nullptr, stream);
}

extern "C" int pl_norm_rope_append(int32_t dtype, int32_t cache_dtype, const void* q, const int64_t* q_strides,
    const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides, void* q_out,
    void* k_out, void* key_cache, const int64_t* key_strides, void* value_cache,
    const int64_t* value_strides, int32_t num_pages, int32_t page_size, const int32_t* page_table,
    int64_t table_ld, int32_t max_pages, const int32_t* past_lens, const int32_t* seq_lens, int32_t rows,
    int32_t row_len, int32_t heads, int32_t kv_heads, int32_t dim, const float* cos, const float* sin,
    int32_t positions, int32_t rot, int32_t interleaved, const float* k_scale, const float* v_scale,
    const void* q_norm, const void* k_norm, int32_t norm_dtype,
    float eps, const int32_t* depths, int64_t depths_ld, void* stream) {
  const char* what = "pl_norm_rope_append";
  if ((q_norm || k_norm) && norm_dtype != PL_F32 && norm_dtype != dtype) {
    pl_set_error("%s: the norms' weights are fp32 or of the model's type (got %d)", what, norm_dtype);
    return PL_ERR_ARG;
  }
  if ((q_norm || k_norm) && !(eps > 0.f && eps < INFINITY)) {
    pl_set_error("%s: eps must be positive and finite (got %g)", what, (double)eps);
    return PL_ERR_ARG;
  }
  norm_args n = {q_norm, k_norm, norm_dtype == PL_F32, eps, depths, depths_ld, 1};
  return append(what, dtype, cache_dtype, q, q_strides, k, k_strides, v, v_strides, q_out, k_out, key_cache, key_strides,
                value_cache, value_strides, num_pages, page_size, page_table, table_ld, max_pages, past_lens, seq_lens,
                rows, row_len, heads, kv_heads, dim, cos, sin, positions, rot, interleaved, k_scale, v_scale, &n, stream);
}
