// Penalties of repeated tokens, biases and grammar masks on logits.
#include "pl_common.h"

// One pass over the logits, 4 at a time (16 bytes of fp32 output, so that a
// wave's stores fill whole lines): memory bounds it (each is read once and
// written once).  A workgroup takes a slice of one row's vocabulary.  What
// is particular to single tokens lies in a table of one LDS word per entry of
// the slice, which the pass reads beside the logits: the workgroup first
// counts the row's history into it (the tokens that fall into the slice;
// integer atomics, the same result in any order) and puts the places of
// biases there.  The history is read again for each slice, from L2, so slices
// are larger for a long one.
namespace {

// A word of the slice's table: how often the token was generated, the place
// plus one of its sum among the slice's biases, whether it was seen at all.
constexpr uint32_t kCountMask = (1u << 20) - 1, kBiasShift = 20, kBiasMask = 0x7ff;
constexpr uint32_t kSeen = 1u << 31;
constexpr int kHistoryMax = (int)kCountMask, kBiasMax = (int)kBiasMask;
constexpr int kVec = 4;     // logits of a thread's load
constexpr int kPasses = 4;  // loads of a thread: its share of the slice
constexpr int kThreadsMax = 1024;
// Places up to the end of the last slice are 32-bit.
constexpr int kVocabMax = INT32_MAX - kThreadsMax * kVec * kPasses;

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

struct penalties {
  float r, f, p;
};

// One logit: its word of the table, the slice's bias sums, its mask bit.
__device__ __forceinline__ float adjust(float x, uint32_t w, const penalties& pen,
                                        const float* sums, bool allowed) {
  if (w & kSeen) {
    x = x > 0.f ? x / pen.r : x * pen.r;
    const uint32_t c = w & kCountMask;
    if (c) x -= pen.f * (float)c + pen.p;
  }
  const int j = (int)((w >> kBiasShift) & kBiasMask);
  if (j) x += sums[j - 1];
  return allowed ? x : -INFINITY;
}

template <int DT, int OT, int THREADS>
__global__ __launch_bounds__(THREADS) void pl_adjust_logits_kernel(logits_args a) {
  typedef typename pl_traits<DT>::T T;
  typedef typename pl_traits<OT>::T O;
  constexpr int kSlice = THREADS * kVec * kPasses;
  __shared__ __attribute__((aligned(16))) uint32_t table[kSlice];
  extern __shared__ __attribute__((aligned(16))) uint32_t dynamic[];  // the slice's biases: ids, values, sums
  __shared__ int s_biases;
  const int b = (int)(blockIdx.x / a.slices), tid = (int)threadIdx.x;
  const int lo = (int)(blockIdx.x % a.slices) * kSlice, hi = min(lo + kSlice, a.vocab);
  const T* in = (const T*)a.logits + b * a.ld;
  O* out = (O*)a.out + b * a.ld_out;
  // Rows have the alignment of their elements alone.  16-bit logits are widened
  // at their load, whose branch then waits for it; fp32's are all in flight.
  T x[kPasses][kVec];
  uint32_t mask[kPasses];
  const uint8_t* allowed = reinterpret_cast<const uint8_t*>(a.allowed + b * a.ld_allowed);
#pragma unroll
  for (int k = 0; k < kPasses; ++k) {
    const int v = lo + (k * THREADS + tid) * kVec;
    if (v + kVec <= hi) __builtin_memcpy(x[k], in + v, sizeof(x[k]));
    mask[k] = a.allowed && v < hi ? allowed[v >> 3] : 0xff;
  }
  // kBatch tokens of the history, THREADS apart, from i on (the last one again
  // past its end).
  constexpr int kBatch = 4;
  int64_t id[kBatch];
  auto look = [&](int i, int end) {
    if (a.wide_tokens) {
      const int64_t* p = (const int64_t*)a.tokens + b * a.ld_tokens;
#pragma unroll
      for (int j = 0; j < kBatch; ++j) id[j] = p[min(i + j * THREADS, end - 1)];
    } else {
      const int32_t* p = (const int32_t*)a.tokens + b * a.ld_tokens;
#pragma unroll
      for (int j = 0; j < kBatch; ++j) id[j] = p[min(i + j * THREADS, end - 1)];
    }
  };
  // The first of them are asked for beside their number: the list is there
  // whole, and what lies beyond `lens` is not counted.
  if (a.tokens && a.history > 0) look(tid, a.history);
  penalties pen;
  pen.r = a.repetition ? a.repetition[b] : 1.f;
  pen.f = a.frequency ? a.frequency[b] : 0.f;
  pen.p = a.presence ? a.presence[b] : 0.f;
  const int n = a.tokens ? min(max(a.lens[b], 0), a.history) : 0;
  const int prompt = a.prompt_lens ? a.prompt_lens[b] : 0;
  const bool special = a.tokens || a.n_bias > 0;
  const int room = (a.n_bias + 3) & ~3;
  int* ids = reinterpret_cast<int*>(dynamic);
  float* values = reinterpret_cast<float*>(dynamic + room);
  float* sums = reinterpret_cast<float*>(dynamic + 2 * room);
  if (special) {
    for (int i = tid; i < kSlice / 4; i += THREADS)
      reinterpret_cast<pl_u32x4*>(table)[i] = pl_u32x4{0, 0, 0, 0};
    if (a.n_bias > 0 && tid < 64) {
      // one wave puts the slice's biases together in the list's order
      constexpr int kLook = 4;  // 64 entries each, asked for at once
      const int32_t* list = a.bias_ids + b * a.ld_bias;
      const float* list_values = a.bias_values + b * a.ld_bias;
      int count = 0;
      for (int j0 = 0; j0 < a.n_bias; j0 += 64 * kLook) {
        int entry[kLook];
        float value[kLook];
#pragma unroll
        for (int k = 0; k < kLook; ++k) {
          const int j = j0 + 64 * k + tid;
          entry[k] = j < a.n_bias ? list[j] : -1;
          value[k] = j < a.n_bias ? list_values[j] : 0.f;
        }
#pragma unroll
        for (int k = 0; k < kLook; ++k) {
          const bool mine = entry[k] >= lo && entry[k] < hi;
          const uint64_t all = __ballot(mine);
          if (mine) {
            const int at = count + __popcll(all & ((1ull << tid) - 1));
            ids[at] = entry[k], values[at] = value[k];
          }
          count += __popcll(all);
        }
      }
      if (tid == 0) s_biases = count;
    }
    __syncthreads();
    for (int i0 = tid; i0 < n; i0 += kBatch * THREADS) {
      if (i0 != tid) look(i0, n);
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int i = i0 + j * THREADS;
        if (i >= n || id[j] < lo || id[j] >= hi) continue;
        if (i >= prompt) atomicAdd(&table[id[j] - lo], 1u);
        atomicOr(&table[id[j] - lo], kSeen);
      }
    }
    if (a.n_bias > 0) {
      // an id's first entry sums all of them, in order; four to a look
      const int count = s_biases;
      for (int j = tid; j < count; j += THREADS) {
        const int id0 = ids[j];
        bool first = true;
        float sum = 0.f;
        for (int i = 0; i < count; i += 4) {
          int look[4];
          float add[4];
          __builtin_memcpy(look, __builtin_assume_aligned(ids + i, 16), 16);
          __builtin_memcpy(add, __builtin_assume_aligned(values + i, 16), 16);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const bool same = i + e < count && look[e] == id0;
            first = first && !(same && i + e < j);
            sum += same ? add[e] : 0.f;
          }
        }
        sums[j] = sum;
        if (first) atomicOr(&table[id0 - lo], (uint32_t)(j + 1) << kBiasShift);
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < kPasses; ++k) {
    const int v = lo + (k * THREADS + tid) * kVec;
    if (v >= hi) break;
    const uint32_t may = mask[k] >> (v & 4);
    uint32_t w[kVec] = {};
    if (special) __builtin_memcpy(w, __builtin_assume_aligned(&table[v - lo], 16), sizeof(w));
    if (v + kVec <= hi) {
      typedef O OV __attribute__((ext_vector_type(kVec), aligned(sizeof(O))));
      OV y;
#pragma unroll
      for (int e = 0; e < kVec; ++e) y[e] = (O)adjust((float)x[k][e], w[e], pen, sums, may >> e & 1);
      // past the caches: the output is read by another launch, whole (256 rows: 41 -> 31 us)
      __builtin_nontemporal_store(y, reinterpret_cast<OV*>(out + v));
    } else {
      for (int e = 0; v + e < hi; ++e)
        out[v + e] = (O)adjust((float)in[v + e], special ? table[v - lo + e] : 0u, pen, sums,
                               may >> e & 1);
    }
  }
}

// Threads of a workgroup, each with kVec * kPasses logits.  Small slices put a
// small batch on more CUs and cost nothing while the history is short; a long
// one is read less often by large slices (32 rows, 8000 tokens: 12.0 -> 9.9
// us; 256 rows, 2000 tokens: 41 us either way).
constexpr int kLongHistory = 4096;

template <int DT, int OT>
int launch(logits_args a, hipStream_t s) {
  const int threads = a.history > kLongHistory ? kThreadsMax : 256;
  const int slice = threads * kVec * kPasses;
  a.slices = (a.vocab + slice - 1) / slice;
  const int64_t blocks = (int64_t)a.rows * a.slices;
  if (!pl_grid_fits(blocks, threads)) {
    pl_set_error("pl_adjust_logits: too many rows (%d)", a.rows);
    return PL_ERR_LIMIT;
  }
  const dim3 grid((unsigned)blocks);
  const size_t lds = (size_t)((a.n_bias + 3) & ~3) * 12;
  if (threads == kThreadsMax)
    pl_adjust_logits_kernel<DT, OT, kThreadsMax><<<grid, kThreadsMax, lds, s>>>(a);
  else
    pl_adjust_logits_kernel<DT, OT, 256><<<grid, 256, lds, s>>>(a);
  return pl_launch_status("pl_adjust_logits");
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
  if (vocab > kVocabMax) {
    pl_set_error("pl_adjust_logits: at most %d logits a row (got %d)", kVocabMax, vocab);
    return PL_ERR_LIMIT;
  }
  if (rows == 0 || vocab == 0) return PL_OK;
  if (!logits || !out || (tokens && (!lens || (token_bytes != 4 && token_bytes != 8))) ||
      (n_bias > 0 && (!bias_ids || !bias_values))) {
    pl_set_error("pl_adjust_logits: null pointer, or tokens of %d bytes", token_bytes);
    return PL_ERR_ARG;
  }
  if (rows > 1 && ld_out < vocab) {
    pl_set_error("pl_adjust_logits: rows of out %lld elements apart overlap (vocab %d)",
                 (long long)ld_out, vocab);
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
  a.n_bias = n_bias, a.wide_tokens = token_bytes == 8;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == PL_F32) return launch<PL_F32, PL_F32>(a, s);
  if (dtype == PL_BF16)
    return out_dtype == PL_F32 ? launch<PL_BF16, PL_F32>(a, s) : launch<PL_BF16, PL_BF16>(a, s);
  return out_dtype == PL_F32 ? launch<PL_F16, PL_F32>(a, s) : launch<PL_F16, PL_F16>(a, s);
}
