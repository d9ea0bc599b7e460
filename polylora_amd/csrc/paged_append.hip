// Rotation by position and append to a paged key-value cache.
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
  if (num_pages < 0 || max_pages < 0 || table_ld < max_pages ||
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
    for (int i = 0; i < 3; ++i) ok = ok && key_strides[i] % e == 0 && value_strides[i] % e == 0;
    if (!ok) {
      pl_set_error("%s: cache pointers and strides must be whole 16-byte pieces", what);
      return PL_ERR_ALIGN;
    }
  }
  return PL_OK;
}

namespace {

constexpr int kThreads = 256;

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
};

// x as stored: rounded to the cache's type, e4m3 after division by the scale
// and saturated (NaN stays NaN).
template <int CT>
__device__ __forceinline__ typename pl_cache_elem<CT>::T to_cache(float x, float scale) {
  if constexpr (CT == PL_F8E4M3) {
    const float y = x / scale;
    const float c = y != y ? y : fminf(fmaxf(y, -kE4M3Max), kE4M3Max);
    return (uint8_t)(__builtin_amdgcn_cvt_pk_fp8_f32(c, c, 0, false) & 0xff);
  } else {
    return (typename pl_cache_elem<CT>::T)x;
  }
}

// One workgroup per token: its threads walk the elements of q, k and v.
template <int DT, int CT>
__global__ __launch_bounds__(kThreads) void pl_rope_append_kernel(append_args a) {
  typedef typename pl_traits<DT>::T T;
  typedef typename pl_cache_elem<CT>::T C;
  const int b = (int)(blockIdx.x / a.row_len), t = (int)(blockIdx.x % a.row_len);
  const int n = a.seq_lens ? min(a.seq_lens[b], a.row_len) : a.row_len;
  const int64_t pos = (int64_t)a.past[b] + t;
  const int64_t column = pos >> a.table.page_shift;
  int page = -1;
  if (t < n && pos >= 0 && pos < a.positions && column < a.table.max_pages)
    page = a.table.p[b * a.table.ld + column];
  const bool live = page >= 0 && page < a.table.num_pages;
  const int64_t slot = pos & ((1 << a.table.page_shift) - 1);
  const int all = (a.heads + 2 * a.kv_heads) * a.dim;
  for (int i = (int)threadIdx.x; i < all; i += kThreads) {
    const int h = i / a.dim, d = i % a.dim;
    const bool is_q = h < a.heads, is_k = !is_q && h < a.heads + a.kv_heads;
    const int hh = is_q ? h : is_k ? h - a.heads : h - a.heads - a.kv_heads;
    const T* x = is_q   ? (const T*)a.q + b * a.qs[0] + t * a.qs[1] + hh * a.qs[2]
                 : is_k ? (const T*)a.k + b * a.ks[0] + t * a.ks[1] + hh * a.ks[2]
                        : (const T*)a.v + b * a.vs[0] + t * a.vs[1] + hh * a.vs[2];
    float y = 0.f;
    if (live) {
      y = (float)x[d];
      if ((is_q || is_k) && d < 2 * a.half) {
        const int p = a.interleaved ? d >> 1 : d % a.half;
        const bool second = a.interleaved ? (d & 1) : d >= a.half;
        const int other = a.interleaved ? d ^ 1 : second ? d - a.half : d + a.half;
        const float c = a.cos[pos * a.half + p], s = a.sin[pos * a.half + p], z = (float)x[other];
        y = second ? y * c + z * s : y * c - z * s;
      }
    }
    const int64_t token = (int64_t)b * a.row_len + t;
    if (is_q) {
      ((T*)a.q_out)[(token * a.heads + hh) * a.dim + d] = (T)y;
    } else {
      const pl_cache_view& cache = is_k ? a.key : a.value;
      if (live)
        ((C*)cache.p)[page * cache.s_page + hh * cache.s_head + slot * cache.s_slot + d] =
            to_cache<CT>(y, CT == PL_F8E4M3 ? (is_k ? a.k_scale : a.v_scale)[hh] : 1.f);
      if (is_k && a.k_out) ((T*)a.k_out)[(token * a.kv_heads + hh) * a.dim + d] = (T)y;
    }
  }
}

}  // namespace

extern "C" int pl_rope_append(int32_t dtype, int32_t cache_dtype, const void* q,
                              const int64_t* q_strides, const void* k, const int64_t* k_strides,
                              const void* v, const int64_t* v_strides, void* q_out, void* k_out,
                              void* key_cache, const int64_t* key_strides, void* value_cache,
                              const int64_t* value_strides, int32_t num_pages, int32_t page_size,
                              const int32_t* page_table, int64_t table_ld, int32_t max_pages,
                              const int32_t* past_lens, const int32_t* seq_lens, int32_t rows,
                              int32_t row_len, int32_t heads, int32_t kv_heads, int32_t dim,
                              const float* cos, const float* sin, int32_t positions, int32_t rot,
                              int32_t interleaved, const float* k_scale, const float* v_scale,
                              void* stream) {
  const int rc = pl_check_paged("pl_rope_append", dtype, cache_dtype, key_cache, key_strides,
                                value_cache, value_strides, num_pages, page_size, page_table,
                                table_ld, max_pages, rows, heads, kv_heads, dim, k_scale, v_scale);
  if (rc) return rc;
  if (row_len < 0 || rot < 0 || rot > dim || rot % 2 != 0 || positions < 0) {
    pl_set_error("pl_rope_append: bad sizes (row_len %d, rot %d of %d, positions %d)", row_len, rot,
                 dim, positions);
    return PL_ERR_ARG;
  }
  const int64_t tokens = (int64_t)rows * row_len;
  if (tokens == 0) return PL_OK;
  if (!q || !k || !v || !q_out || !q_strides || !k_strides || !v_strides || !past_lens ||
      (rot > 0 && positions > 0 && (!cos || !sin))) {
    pl_set_error("pl_rope_append: null pointer");
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
      pl_set_error("pl_rope_append: an output overlaps an input");
      return PL_ERR_ARG;
    }
  if (!pl_grid_fits(tokens, kThreads)) {
    pl_set_error("pl_rope_append: too many tokens (%lld)", (long long)tokens);
    return PL_ERR_LIMIT;
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
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)tokens);
  if (cache_dtype == PL_F8E4M3) {
    if (dtype == PL_BF16)
      pl_rope_append_kernel<PL_BF16, PL_F8E4M3><<<grid, kThreads, 0, s>>>(a);
    else
      pl_rope_append_kernel<PL_F16, PL_F8E4M3><<<grid, kThreads, 0, s>>>(a);
  } else if (dtype == PL_F32) {
    pl_rope_append_kernel<PL_F32, PL_F32><<<grid, kThreads, 0, s>>>(a);
  } else if (dtype == PL_BF16) {
    pl_rope_append_kernel<PL_BF16, PL_BF16><<<grid, kThreads, 0, s>>>(a);
  } else {
    pl_rope_append_kernel<PL_F16, PL_F16><<<grid, kThreads, 0, s>>>(a);
  }
  return pl_launch_status("pl_rope_append");
}
