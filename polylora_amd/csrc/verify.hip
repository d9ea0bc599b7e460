// Which drafted tokens of a row stay, and the token that follows them.
#include "pl_common.h"

// A row's tokens form a tree: token 0 is the row's last one, the others are drafts,
// each behind its parent.  Token n has logits x and with them the probabilities
//   p_v = e_v / Z,  e_v = exp((x_v - max x) / temperature),  Z = sum_v e_v
// of what follows it.  From token 0 on, the row moves to a child or stops:
//   drafts without probabilities: v is the first with sum_{i <= v} e_i > u Z; the
//     row moves to the child that holds v, or stops with v;
//   a line of drafts with the probabilities q that they were drawn from: the row
//     moves to the next draft, d, if u q_d < p_d; else it stops with the first v
//     whose sum of max(p_i - q_i, 0) passes u' times the whole sum;
//   temperature 0: v is the first place of the largest logit.
// Weights and sums are 64-bit: a sum of 10^5 weights decides between tokens whose
// borders lie 10^-6 apart and less, and a running sum in fp32 is off by as much.
namespace {

constexpr int kThreads = 1024;
constexpr int kSlice = 4096;     // logits whose weights are summed apart
constexpr int kSlicesMax = 2048;

struct verify_args {
  const void* logits;
  int64_t ld_row, ld_node;
  const void* tokens;
  int64_t ld_tokens;
  const float* uniforms;
  int64_t ld_uniforms;
  const int32_t* parents;  // null for a line
  int64_t ld_parents;
  const float* draft_probs;  // of the drafts behind token n; null where drafts have none
  int64_t ld_draft_row, ld_draft_node;
  const float* temperature;
  const int32_t* seq_lens;
  int32_t* path;     // [rows][nodes]
  int32_t* counts;   // [rows]
  int64_t* next;     // [rows]
  int32_t rows, nodes, vocab, wide_tokens, slices;
};

// 2^t for t <= 0, to 2e-13: the power of two of the nearest integer times the
// exponential's series for the rest.
__device__ __forceinline__ double exp2_64(double t) {
  const double n = __builtin_rint(t);
  const double f = (t - n) * 0.69314718055994530942;
  double p = 1.0 / 39916800.0;
  p = fma(p, f, 1.0 / 3628800.0);
  p = fma(p, f, 1.0 / 362880.0);
  p = fma(p, f, 1.0 / 40320.0);
  p = fma(p, f, 1.0 / 5040.0);
  p = fma(p, f, 1.0 / 720.0);
  p = fma(p, f, 1.0 / 120.0);
  p = fma(p, f, 1.0 / 24.0);
  p = fma(p, f, 1.0 / 6.0);
  p = fma(p, f, 0.5);
  p = fma(p, f, 1.0);
  p = fma(p, f, 1.0);
  return __builtin_ldexp(p, (int)n);
}

// The weight of a logit beside the largest, `per` = log2(e) / temperature.  -inf
// gives 0, NaN gives NaN.
__device__ __forceinline__ double weight(float x, float top, double per) {
  const double t = ((double)x - (double)top) * per;
  return t < -1000.0 ? 0.0 : t != t ? t : exp2_64(t);
}

template <typename V, typename Op>
__device__ __forceinline__ V block_all(V x, V* shared, Op op) {
  const int tid = (int)threadIdx.x;
  for (int d = 1; d < 64; d *= 2) x = op(x, __shfl_xor(x, d));
  __syncthreads();
  if ((tid & 63) == 0) shared[tid >> 6] = x;
  __syncthreads();
  V r = shared[0];
  for (int w = 1; w < kThreads / 64; ++w) r = op(r, shared[w]);
  return r;
}

// A workgroup walks one row.
template <int DT>
__global__ __launch_bounds__(kThreads) void pl_verify_tokens_kernel(verify_args a) {
  typedef typename pl_traits<DT>::T T;
  __shared__ double s_sum[kSlicesMax];
  __shared__ double s_red[kThreads / 64];
  __shared__ float s_top[kThreads / 64];
  __shared__ int s_int[kThreads / 64];
  const int b = (int)blockIdx.x, tid = (int)threadIdx.x;
  const int n = a.seq_lens ? min(a.seq_lens[b], a.nodes) : a.nodes;
  const float heat = a.temperature ? a.temperature[b] : 1.f;
  const bool greedy = heat == 0.f;
  const double per = 1.44269504088896340736 / (double)heat;
  auto token_of = [&](int i) -> int64_t {
    return a.wide_tokens ? ((const int64_t*)a.tokens)[b * a.ld_tokens + i]
                         : ((const int32_t*)a.tokens)[b * a.ld_tokens + i];
  };
  int32_t* path = a.path + (int64_t)b * a.nodes;
  for (int i = tid; i < a.nodes; i += kThreads) path[i] = i == 0 && n > 0 ? 0 : -1;
  int node = 0, count = n > 0 ? 1 : 0;
  int64_t token = -1;
  while (n > 0) {
    const T* x = (const T*)a.logits + b * a.ld_row + node * a.ld_node;
    float top = -INFINITY;
    int bad = 0;
    for (int v = tid; v < a.vocab; v += kThreads) {
      const float y = (float)x[v];
      bad |= !(y < INFINITY);
      top = fmaxf(top, y);
    }
    top = block_all(top, s_top, [](float p, float q) { return fmaxf(p, q); });
    bad = block_all(bad, s_int, [](int p, int q) { return p | q; });
    if (bad || top == -INFINITY || !(heat >= 0.f && heat < INFINITY)) {
      token = -1;
      break;
    }
    const bool line = a.draft_probs != nullptr, last = node + 1 >= n;
    const float* q = line && !last ? a.draft_probs + b * a.ld_draft_row + node * a.ld_draft_node : nullptr;
    int best = INT32_MAX;
    double z = 0.0;
    if (greedy) {
      for (int v = tid; v < a.vocab; v += kThreads)
        if ((float)x[v] == top) best = min(best, v);
      best = block_all(best, s_int, [](int p, int r) { return min(p, r); });
    } else {
      for (int v = tid; v < a.vocab; v += kThreads) z += weight((float)x[v], top, per);
      z = block_all(z, s_red, [](double p, double r) { return p + r; });
    }
    const float u = a.uniforms[b * a.ld_uniforms + node];
    if (line && !last) {
      const int64_t d = token_of(node + 1);
      const bool known = d >= 0 && d < a.vocab;
      const bool go = greedy ? d == best
                             : known && (double)u * (double)q[d] * z < weight((float)x[d], top, per);
      if (go) {
        if (tid == 0) path[count] = node + 1;
        ++count, ++node;
        continue;
      }
    }
    if (greedy) {
      token = best;
    } else {
      // draw: sums of slices, then the place inside one
      const float u2 = line ? a.uniforms[b * a.ld_uniforms + n - 1] : u;
      bool rest = q != nullptr;
      auto share = [&](int v) {
        const double e = weight((float)x[v], top, per);
        return rest ? fmax(e - (double)q[v] * z, 0.0) : e;
      };
      double total = 0.0;
      for (int turn = 0; turn < 2; ++turn) {
        total = 0.0;
        for (int s = 0; s < a.slices; ++s) {
          double part = 0.0;
          for (int v = s * kSlice + tid; v < min((s + 1) * kSlice, a.vocab); v += kThreads) part += share(v);
          part = block_all(part, s_red, [](double p, double r) { return p + r; });
          if (tid == 0) s_sum[s] = part;
          total += part;
        }
        __syncthreads();
        if (!rest || total > 0.0) break;
        rest = false;  // the two agree everywhere: draw from p
      }
      const double target = (double)u2 * total;
      double upto = 0.0;
      int s = 0;
      for (; s + 1 < a.slices && upto + s_sum[s] <= target; ++s) upto += s_sum[s];
      // inside the slice: running sums of 1024 at a time
      int found = INT32_MAX, some = -1;
      for (int v0 = s * kSlice; v0 < min((s + 1) * kSlice, a.vocab) && found == INT32_MAX; v0 += kThreads) {
        const int v = v0 + tid;
        const double mine = v < a.vocab ? share(v) : 0.0;
        double run = mine;
        for (int d = 1; d < 64; d *= 2) {
          const double lower = __shfl_up(run, d);
          if ((tid & 63) >= d) run += lower;
        }
        __syncthreads();
        if ((tid & 63) == 63) s_red[tid >> 6] = run;
        __syncthreads();
        double before = upto;
        for (int w = 0; w < tid >> 6; ++w) before += s_red[w];
        for (int w = 0; w < kThreads / 64; ++w) upto += s_red[w];
        found = block_all(mine > 0.0 && before + run > target ? v : INT32_MAX, s_int,
                          [](int p, int r) { return min(p, r); });
        some = max(some, block_all(mine > 0.0 ? v : -1, s_int, [](int p, int r) { return max(p, r); }));
      }
      token = found != INT32_MAX ? found : some;
    }
    if (line) break;
    int child = INT32_MAX;
    for (int c = tid + 1; c < n; c += kThreads) {
      const int parent = a.parents ? a.parents[b * a.ld_parents + c] : c - 1;
      if (parent == node && c > node && token_of(c) == token) child = min(child, c);
    }
    child = block_all(child, s_int, [](int p, int r) { return min(p, r); });
    if (child == INT32_MAX) break;
    if (tid == 0) path[count] = child;
    ++count, node = child;
  }
  if (tid == 0) a.counts[b] = count, a.next[b] = token;
}

}  // namespace

extern "C" int pl_verify_tokens(int32_t dtype, const void* logits, int64_t ld_row, int64_t ld_node,
                                const void* tokens, int32_t token_bytes, int64_t ld_tokens,
                                const float* uniforms, int64_t ld_uniforms, const int32_t* parents,
                                int64_t ld_parents, const float* draft_probs, int64_t ld_draft_row,
                                int64_t ld_draft_node, const float* temperature, const int32_t* seq_lens,
                                int32_t rows, int32_t nodes, int32_t vocab, int32_t* path, int32_t* counts,
                                int64_t* next, void* stream) {
  const char* what = "pl_verify_tokens";
  if (dtype != PL_F32 && dtype != PL_BF16 && dtype != PL_F16) {
    pl_set_error("%s: unknown element type %d", what, dtype);
    return PL_ERR_ARG;
  }
  if (rows < 0 || nodes < 0 || vocab < 0 || (token_bytes != 4 && token_bytes != 8)) {
    pl_set_error("%s: bad sizes (rows %d, nodes %d, vocab %d, tokens of %d bytes)", what, rows, nodes, vocab,
                 token_bytes);
    return PL_ERR_ARG;
  }
  if (vocab > kSlice * kSlicesMax) {
    pl_set_error("%s: at most %d logits to a token (got %d)", what, kSlice * kSlicesMax, vocab);
    return PL_ERR_LIMIT;
  }
  if (parents && draft_probs) {
    pl_set_error("%s: drafts with probabilities form a line, not a tree", what);
    return PL_ERR_ARG;
  }
  if (rows == 0) return PL_OK;
  if (!counts || !next || (nodes > 0 && (!path || !tokens || !uniforms || (vocab > 0 && !logits)))) {
    pl_set_error("%s: null pointer", what);
    return PL_ERR_ARG;
  }
  verify_args a;
  a.logits = logits, a.ld_row = ld_row, a.ld_node = ld_node, a.tokens = tokens, a.ld_tokens = ld_tokens;
  a.uniforms = uniforms, a.ld_uniforms = ld_uniforms, a.parents = parents, a.ld_parents = ld_parents;
  a.draft_probs = draft_probs, a.ld_draft_row = ld_draft_row, a.ld_draft_node = ld_draft_node;
  a.temperature = temperature, a.seq_lens = seq_lens, a.path = path, a.counts = counts, a.next = next;
  a.rows = rows, a.nodes = nodes, a.vocab = vocab, a.wide_tokens = token_bytes == 8;
  a.slices = (vocab + kSlice - 1) / kSlice;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)rows);
  if (!pl_grid_fits(rows, kThreads)) {
    pl_set_error("%s: too many rows (%d)", what, rows);
    return PL_ERR_LIMIT;
  }
  if (dtype == PL_F32)
    pl_verify_tokens_kernel<PL_F32><<<grid, kThreads, 0, s>>>(a);
  else if (dtype == PL_BF16)
    pl_verify_tokens_kernel<PL_BF16><<<grid, kThreads, 0, s>>>(a);
  else
    pl_verify_tokens_kernel<PL_F16><<<grid, kThreads, 0, s>>>(a);
  return pl_launch_status(what);
}
