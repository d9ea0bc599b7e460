// Penalties of repeated tokens, biases and grammar masks on logits.
#include "pl_common.h"

namespace {

constexpr int kThreads = 256;
// Vocabulary entries of one workgroup: a word of LDS for each.
constexpr int kSlice = 4096;
// A word of the slice's table: how often the token was generated, the place
// plus one of its first entry in the bias list, whether it was seen at all.
constexpr uint32_t kCountMask = (1u << 20) - 1, kBiasShift = 20, kBiasMask = 0x7ff;
constexpr uint32_t kSeen = 1u << 31;
constexpr int kHistoryMax = (int)kCountMask, kBiasMax = (int)kBiasMask;

struct logits_args {
  const void* logits;
  void* out;
  const void* tokens;
  const int32_t *lens, *prompt_lens;
  const float *repetition, *presence, *frequency;
  const int32_t* bias_ids;
  const float* bias_values;
  const int32_t* allowed;
  int64_t ld, ld_out, ld_tokens, ld_bias, ld_allowed;
  int32_t rows, vocab, history, n_bias, wide_tokens, slices;
};

// One workgroup per (row, slice of the vocabulary): it counts the row's
// history and looks up its biases in LDS, then walks its logits once.
template <int DT, int OT>
__global__ __launch_bounds__(kThreads) void pl_adjust_logits_kernel(logits_args a) {
  typedef typename pl_traits<DT>::T T;
  typedef typename pl_traits<OT>::T O;
  __shared__ uint32_t table[kSlice];
  const int b = (int)(blockIdx.x / a.slices), tid = (int)threadIdx.x;
  const int lo = (int)(blockIdx.x % a.slices) * kSlice, hi = min(lo + kSlice, a.vocab);
  for (int i = tid; i < kSlice; i += kThreads) table[i] = 0;
  __syncthreads();
  const int n = a.tokens ? min(max(a.lens[b], 0), a.history) : 0;
  const int prompt = a.prompt_lens ? a.prompt_lens[b] : 0;
  for (int i = tid; i < n; i += kThreads) {
    const int64_t id = a.wide_tokens ? ((const int64_t*)a.tokens)[b * a.ld_tokens + i]
                                     : ((const int32_t*)a.tokens)[b * a.ld_tokens + i];
    if (id < lo || id >= hi) continue;
    atomicOr(&table[id - lo], kSeen);
    if (i >= prompt) atomicAdd(&table[id - lo], 1u);
  }
  const int32_t* ids = a.bias_ids + b * a.ld_bias;
  const float* values = a.bias_values + b * a.ld_bias;
  for (int j = tid; j < a.n_bias; j += kThreads) {
    const int id = ids[j];
    if (id < lo || id >= hi) continue;
    bool first = true;
    for (int i = 0; i < j; ++i) first = first && ids[i] != id;
    if (first) atomicOr(&table[id - lo], (uint32_t)(j + 1) << kBiasShift);
  }
  __syncthreads();
  const float r = a.repetition ? a.repetition[b] : 1.f;
  const float f = a.frequency ? a.frequency[b] : 0.f, p = a.presence ? a.presence[b] : 0.f;
  for (int v = lo + tid; v < hi; v += kThreads) {
    float x = (float)((const T*)a.logits)[b * a.ld + v];
    const uint32_t w = table[v - lo];
    if (w & kSeen) {
      x = x > 0.f ? x / r : x * r;
      const uint32_t c = w & kCountMask;
      if (c) x -= f * (float)c + p;
    }
    const int j = (int)((w >> kBiasShift) & kBiasMask);
    if (j) {
      float bias = 0.f;
      for (int i = j - 1; i < a.n_bias; ++i)
        if (ids[i] == v) bias += values[i];
      x += bias;
    }
    if (a.allowed && !((uint32_t)a.allowed[b * a.ld_allowed + (v >> 5)] >> (v & 31) & 1))
      x = -INFINITY;
    ((O*)a.out)[b * a.ld_out + v] = (O)x;
  }
}

}  // namespace

extern "C" int pl_adjust_logits(int32_t dtype, int32_t out_dtype, const void* logits, int64_t ld,
                                void* out, int64_t ld_out, int32_t rows, int32_t vocab,
                                const void* tokens, int32_t token_bytes, int64_t ld_tokens,
                                int32_t history, const int32_t* lens, const int32_t* prompt_lens,
                                const float* repetition, const float* presence,
                                const float* frequency, const int32_t* bias_ids,
                                const float* bias_values, int64_t ld_bias, int32_t n_bias,
                                const int32_t* allowed, int64_t ld_allowed, void* stream) {
  if ((dtype != PL_F32 && dtype != PL_BF16 && dtype != PL_F16) ||
      (out_dtype != PL_F32 && out_dtype != dtype)) {
    pl_set_error("pl_adjust_logits: logits of type %d to type %d", dtype, out_dtype);
    return PL_ERR_ARG;
  }
  if (rows < 0 || vocab < 0 || history < 0 || n_bias < 0) {
    pl_set_error("pl_adjust_logits: negative size (rows %d, vocab %d, history %d, biases %d)", rows,
                 vocab, history, n_bias);
    return PL_ERR_ARG;
  }
  if (history > kHistoryMax || n_bias > kBiasMax) {
    pl_set_error("pl_adjust_logits: at most %d tokens of history and %d biases (got %d and %d)",
                 kHistoryMax, kBiasMax, history, n_bias);
    return PL_ERR_LIMIT;
  }
  if (rows == 0 || vocab == 0) return PL_OK;
  if (!logits || !out || (tokens && (!lens || (token_bytes != 4 && token_bytes != 8))) ||
      (n_bias > 0 && (!bias_ids || !bias_values))) {
    pl_set_error("pl_adjust_logits: null pointer, or tokens of %d bytes", token_bytes);
    return PL_ERR_ARG;
  }
  const int64_t in_bytes = ((rows - 1) * ld + vocab) * pl_elem_size(dtype);
  const int64_t out_bytes = ((rows - 1) * ld_out + vocab) * pl_elem_size(out_dtype);
  if (pl_ranges_meet(logits, in_bytes, out, out_bytes) &&
      !(logits == out && dtype == out_dtype && (ld == ld_out || rows == 1))) {
    pl_set_error("pl_adjust_logits: out overlaps the logits without being them");
    return PL_ERR_ARG;
  }
  logits_args a;
  a.logits = logits, a.out = out, a.tokens = tokens, a.lens = lens, a.prompt_lens = prompt_lens;
  a.repetition = repetition, a.presence = presence, a.frequency = frequency;
  a.bias_ids = bias_ids, a.bias_values = bias_values, a.allowed = allowed;
  a.ld = ld, a.ld_out = ld_out, a.ld_tokens = ld_tokens, a.ld_bias = ld_bias;
  a.ld_allowed = ld_allowed, a.rows = rows, a.vocab = vocab, a.history = history;
  a.n_bias = n_bias, a.wide_tokens = token_bytes == 8, a.slices = (vocab + kSlice - 1) / kSlice;
  const int64_t blocks = (int64_t)rows * a.slices;
  if (!pl_grid_fits(blocks, kThreads)) {
    pl_set_error("pl_adjust_logits: too many rows (%d)", rows);
    return PL_ERR_LIMIT;
  }
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)blocks);
  if (dtype == PL_F32)
    pl_adjust_logits_kernel<PL_F32, PL_F32><<<grid, kThreads, 0, s>>>(a);
  else if (dtype == PL_BF16 && out_dtype == PL_F32)
    pl_adjust_logits_kernel<PL_BF16, PL_F32><<<grid, kThreads, 0, s>>>(a);
  else if (dtype == PL_BF16)
    pl_adjust_logits_kernel<PL_BF16, PL_BF16><<<grid, kThreads, 0, s>>>(a);
  else if (out_dtype == PL_F32)
    pl_adjust_logits_kernel<PL_F16, PL_F32><<<grid, kThreads, 0, s>>>(a);
  else
    pl_adjust_logits_kernel<PL_F16, PL_F16><<<grid, kThreads, 0, s>>>(a);
  return pl_launch_status("pl_adjust_logits");
}
