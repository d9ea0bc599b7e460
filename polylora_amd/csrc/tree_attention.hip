// Attention of drafted tokens over a paged key-value cache and over one another.
//
// Token i of row b looks at the row's tokens before the drafts (the last `window` of
// them counted from its own depth) and at those drafts that its mask names, itself
// among them:
//   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  s_j = scale * q . k_j,  m = max_j s_j.
#include "pl_paged.h"

namespace {

constexpr int kThreads = 256;

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
  float scale;
  int32_t rows, row_len, heads, kv_heads, dim, window;
};

template <int DT, int CT>
__device__ __forceinline__ float element(const void* p, int64_t at) {
  if constexpr (CT == PL_F8E4M3)
    return __builtin_amdgcn_cvt_f32_fp8(((const uint8_t*)p)[at], 0);
  else
    return (float)((const typename pl_traits<DT>::T*)p)[at];
}

// A wave for each (row, token, head): a lane for a key, then for elements of the values.
template <int DT, int CT>
__global__ __launch_bounds__(kThreads) void pl_tree_attention_kernel(tree_args a) {
  typedef typename pl_traits<DT>::T T;
  __shared__ float s_q[kThreads / 64][kHeadDimMax];
  const int wave = (int)threadIdx.x >> 6, lane = (int)threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * (kThreads / 64) + wave;
  if (item >= (int64_t)a.rows * a.row_len * a.heads) return;
  const int h = (int)(item % a.heads), i = (int)(item / a.heads % a.row_len);
  const int b = (int)(item / a.heads / a.row_len);
  const int hk = h / (a.heads / a.kv_heads);
  const int n = min(a.seq_lens ? a.seq_lens[b] : a.row_len, a.row_len);
  const int64_t past = a.past[b];
  const int64_t cap = a.table.num_pages ? (int64_t)a.table.max_pages << a.table.page_shift : 0;
  const int64_t len = i < n && past >= 0 ? min(past + n, cap) : 0;
  const int depth = a.depths && i < n ? a.depths[b * a.depths_row + i] : i;
  const int64_t first = a.window > 0 ? max((int64_t)0, past + depth - a.window + 1) : 0;
  const T* q = (const T*)a.q + b * a.q_row + i * a.q_token + h * a.q_head;
  for (int d = lane; d < a.dim; d += 64) s_q[wave][d] = (float)q[d];
  float m = -INFINITY, l = 0.f, o[kHeadDimMax / 64] = {};
  const float k_scale = CT == PL_F8E4M3 ? a.k_scale[hk] : 1.f, v_scale = CT == PL_F8E4M3 ? a.v_scale[hk] : 1.f;
  for (int64_t j0 = a.visible ? min(first, past) : first; j0 < len; j0 += 64) {
    const int64_t j = j0 + lane;
    int page = -1;
    if (j < len) {
      bool seen = j >= first;
      if (j >= past) {
        const int t = (int)(j - past);
        seen = a.visible ? a.visible[b * a.visible_row + i * a.visible_token + (t >> 5)] >> (t & 31) & 1
                         : seen && t <= i;
      }
      if (seen) page = a.table.p[b * a.table.ld + (j >> a.table.page_shift)];
      if (page >= a.table.num_pages) page = -1;
    }
    const int64_t slot = j & ((1 << a.table.page_shift) - 1);
    float s = -INFINITY;
    if (page >= 0) {
      const int64_t at = page * a.key.s_page + hk * a.key.s_head + slot * a.key.s_slot;
      s = 0.f;
      for (int d = 0; d < a.dim; ++d) s = fmaf(s_q[wave][d], element<DT, CT>(a.key.p, at + d), s);
      s *= a.scale * k_scale;
    }
    float top = s;
    for (int d = 1; d < 64; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
    top = fmaxf(top, m);
    const float ref = top == -INFINITY ? 0.f : top, keep = expf(m - ref);
    m = top, l *= keep;
    const float p = expf(s - ref);
    l += p;
    for (int k = 0; k < kHeadDimMax / 64; ++k) o[k] *= keep;
    const int64_t at = page * a.value.s_page + hk * a.value.s_head + slot * a.value.s_slot;
    for (int t = 0; t < 64; ++t) {
      if (__shfl(page, t) < 0) continue;
      const float pt = __shfl(p, t);
      const int64_t from = __shfl(at, t);
      for (int k = 0; k * 64 + lane < a.dim; ++k) o[k] += pt * element<DT, CT>(a.value.p, from + k * 64 + lane);
    }
  }
  for (int d = 1; d < 64; d *= 2) l += __shfl_xor(l, d);
  T* out = (T*)a.out + item * a.dim;
  for (int k = 0; k * 64 + lane < a.dim; ++k) out[k * 64 + lane] = (T)(l == 0.f ? 0.f : o[k] / l * v_scale);
}

template <int DT, int CT>
int launch(const tree_args& a, hipStream_t s) {
  const int64_t items = (int64_t)a.rows * a.row_len * a.heads, blocks = (items + kThreads / 64 - 1) / (kThreads / 64);
  if (!pl_grid_fits(blocks, kThreads)) {
    pl_set_error("pl_tree_attention: too many tokens (%lld)", (long long)a.rows * a.row_len);
    return PL_ERR_LIMIT;
  }
  pl_tree_attention_kernel<DT, CT><<<dim3((unsigned)blocks), kThreads, 0, s>>>(a);
  return pl_launch_status("pl_tree_attention");
}

}  // namespace

extern "C" int pl_tree_attention(int32_t dtype, int32_t cache_dtype, const void* q, const int64_t* q_strides,
                                 const void* key_cache, const int64_t* key_strides, const void* value_cache,
                                 const int64_t* value_strides, int32_t num_pages, int32_t page_size,
                                 const int32_t* page_table, int64_t table_ld, int32_t max_pages,
                                 const int32_t* past_lens, const int32_t* seq_lens, const int32_t* visible,
                                 int64_t visible_row, int64_t visible_token, int32_t words, const int32_t* depths,
                                 int64_t depths_row, int32_t rows, int32_t row_len, int32_t heads, int32_t kv_heads,
                                 int32_t dim, float scale, int32_t window, const float* k_scale, const float* v_scale,
                                 void* out, void* stream) {
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
  tree_args a;
  a.q = q, a.q_row = q_strides[0], a.q_token = q_strides[1], a.q_head = q_strides[2];
  a.key = {const_cast<void*>(key_cache), key_strides[0], key_strides[1], key_strides[2]};
  a.value = {const_cast<void*>(value_cache), value_strides[0], value_strides[1], value_strides[2]};
  a.table = {page_table, table_ld, max_pages, num_pages, pl_log2_exact(page_size)};
  a.past = past_lens, a.seq_lens = seq_lens, a.visible = visible, a.visible_row = visible_row;
  a.visible_token = visible_token, a.depths = visible ? depths : nullptr, a.depths_row = depths_row;
  a.k_scale = k_scale, a.v_scale = v_scale, a.out = out, a.scale = scale, a.rows = rows, a.row_len = row_len;
  a.heads = heads, a.kv_heads = kv_heads, a.dim = dim, a.window = window;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (cache_dtype == PL_F8E4M3)
    return dtype == PL_BF16 ? launch<PL_BF16, PL_F8E4M3>(a, s) : launch<PL_F16, PL_F8E4M3>(a, s);
  if (dtype == PL_F32) return launch<PL_F32, PL_F32>(a, s);
  return dtype == PL_BF16 ? launch<PL_BF16, PL_BF16>(a, s) : launch<PL_F16, PL_F16>(a, s);
}
