// Attention of one new token per row over a paged key-value cache.
#include "pl_paged.h"

namespace {

constexpr int kWaves = 4;

struct attend_args {
  const void* q;
  int64_t q_row, q_head;
  pl_cache_view key, value;
  pl_page_table table;
  const int32_t* lens;
  const float *k_scale, *v_scale;
  void* out;  // contiguous [rows][heads][dim]
  float scale;
  int32_t rows, heads, kv_heads, dim, window;
};

template <int CT>
__device__ __forceinline__ float from_cache(typename pl_cache_elem<CT>::T x) {
  if constexpr (CT == PL_F8E4M3)
    return __builtin_amdgcn_cvt_f32_fp8((int)x, 0);
  else
    return (float)x;
}

// One workgroup per (row, query head).  Each wave walks every kWaves-th token
// with a running maximum, sum and output of its own, its lanes holding dim / 64
// elements each; the waves' are joined in LDS at the end.
template <int DT, int CT>
__global__ __launch_bounds__(kWaves * 64) void pl_paged_attention_kernel(attend_args a) {
  typedef typename pl_traits<DT>::T T;
  typedef typename pl_cache_elem<CT>::T C;
  constexpr int kPer = kHeadDimMax / 64;
  const int b = (int)(blockIdx.x / a.heads), h = (int)(blockIdx.x % a.heads);
  const int hk = h / (a.heads / a.kv_heads);
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  const int64_t cap = (int64_t)a.table.max_pages << a.table.page_shift;
  const int len = (int)min((int64_t)max(a.lens[b], 0), cap);
  const int first = a.window > 0 ? max(0, len - a.window) : 0;
  float q[kPer], o[kPer], m = -INFINITY, l = 0.f;
  const float scale = a.scale * (CT == PL_F8E4M3 ? a.k_scale[hk] : 1.f);
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int d = lane + 64 * i;
    q[i] = d < a.dim ? (float)((const T*)a.q)[b * a.q_row + h * a.q_head + d] * scale : 0.f;
    o[i] = 0.f;
  }
  for (int j = first + wave; j < len; j += kWaves) {
    const int page = a.table.p[b * a.table.ld + (j >> a.table.page_shift)];
    if (page < 0 || page >= a.table.num_pages) continue;
    const int slot = j & ((1 << a.table.page_shift) - 1);
    const C* k = (const C*)a.key.p + page * a.key.s_page + hk * a.key.s_head + slot * a.key.s_slot;
    const C* v =
        (const C*)a.value.p + page * a.value.s_page + hk * a.value.s_head + slot * a.value.s_slot;
    float s = 0.f, x[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int d = lane + 64 * i;
      s += d < a.dim ? q[i] * from_cache<CT>(k[d]) : 0.f;
      x[i] = d < a.dim ? from_cache<CT>(v[d]) : 0.f;
    }
#pragma unroll
    for (int w = 32; w > 0; w >>= 1) s += __shfl_xor(s, w);
    const float top = fmaxf(m, s);
    const float keep = m == top ? 1.f : __expf(m - top), p = s == top ? 1.f : __expf(s - top);
    l = l * keep + p;
#pragma unroll
    for (int i = 0; i < kPer; ++i) o[i] = o[i] * keep + p * x[i];
    m = top;
  }
  __shared__ float s_m[kWaves], s_l[kWaves], s_o[kWaves][kHeadDimMax];
  if (lane == 0) s_m[wave] = m, s_l[wave] = l;
#pragma unroll
  for (int i = 0; i < kPer; ++i) s_o[wave][lane + 64 * i] = o[i];
  __syncthreads();
  const int d = (int)threadIdx.x;
  if (d >= a.dim) return;
  float top = -INFINITY, sum = 0.f, acc = 0.f;
  for (int w = 0; w < kWaves; ++w) top = fmaxf(top, s_m[w]);
  for (int w = 0; w < kWaves; ++w) {
    const float f = s_l[w] > 0.f ? (s_m[w] == top ? 1.f : __expf(s_m[w] - top)) : 0.f;
    sum += f * s_l[w], acc += f * s_o[w][d];
  }
  const float y = sum > 0.f ? acc / sum * (CT == PL_F8E4M3 ? a.v_scale[hk] : 1.f) : sum;
  ((T*)a.out)[((int64_t)b * a.heads + h) * a.dim + d] = (T)y;
}

}  // namespace

extern "C" int pl_paged_attention(int32_t dtype, int32_t cache_dtype, const void* q,
                                  const int64_t* q_strides, const void* key_cache,
                                  const int64_t* key_strides, const void* value_cache,
                                  const int64_t* value_strides, int32_t num_pages,
                                  int32_t page_size, const int32_t* page_table, int64_t table_ld,
                                  int32_t max_pages, const int32_t* lens, int32_t rows,
                                  int32_t heads, int32_t kv_heads, int32_t dim, float scale,
                                  int32_t window, const float* k_scale, const float* v_scale,
                                  void* out, void* stream) {
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
  if (!pl_grid_fits((int64_t)rows * heads, kWaves * 64)) {
    pl_set_error("pl_paged_attention: too many rows (%d)", rows);
    return PL_ERR_LIMIT;
  }
  attend_args a;
  a.q = q, a.q_row = q_strides[0], a.q_head = q_strides[1];
  a.key = {const_cast<void*>(key_cache), key_strides[0], key_strides[1], key_strides[2]};
  a.value = {const_cast<void*>(value_cache), value_strides[0], value_strides[1], value_strides[2]};
  a.table = {page_table, table_ld, max_pages, num_pages, pl_log2_exact(page_size)};
  a.lens = lens, a.k_scale = k_scale, a.v_scale = v_scale, a.out = out, a.scale = scale;
  a.rows = rows, a.heads = heads, a.kv_heads = kv_heads, a.dim = dim, a.window = window;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)(rows * heads));
  if (cache_dtype == PL_F8E4M3) {
    if (dtype == PL_BF16)
      pl_paged_attention_kernel<PL_BF16, PL_F8E4M3><<<grid, kWaves * 64, 0, s>>>(a);
    else
      pl_paged_attention_kernel<PL_F16, PL_F8E4M3><<<grid, kWaves * 64, 0, s>>>(a);
  } else if (dtype == PL_F32) {
    pl_paged_attention_kernel<PL_F32, PL_F32><<<grid, kWaves * 64, 0, s>>>(a);
  } else if (dtype == PL_BF16) {
    pl_paged_attention_kernel<PL_BF16, PL_BF16><<<grid, kWaves * 64, 0, s>>>(a);
  } else {
    pl_paged_attention_kernel<PL_F16, PL_F16><<<grid, kWaves * 64, 0, s>>>(a);
  }
  return pl_launch_status("pl_paged_attention");
}
