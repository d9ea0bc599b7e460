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
//
// A launch looks at all tokens of all rows at once, a wave to each piece of a token's
// logits, which it reads once into registers: the piece's largest, then the sum of
// its weights beside that.  The wave of a token's last piece to end puts the
// sums together and says where the row would go from there; whoever says so
// last for a row follows its tokens.  Where a large batch does not run all at
// once, tokens lie in the grid's order before those behind them, and a workgroup
// leaves out a token that a row is known to have turned away from: what it would
// have found counts for nothing.  Drawing from what is left of p beside q needs
// Z first, and is a second launch, over one token of each row.
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kVec = 4;          // logits of a lane's load
constexpr int kNodesMax = 1024;  // tokens of a row
constexpr int kVocabMax = 1 << 24;
// Loads of a lane to a piece: pieces of 1024 logits for few rows, that all CUs take
// part, of 2048 above kManyPieces of those, whose beginnings and ends cost less.
constexpr int kFewPasses = 4, kManyPasses = 8;
constexpr int kManyPieces = 8192;
// Workgroups above which some end before others begin, so that looking for tokens
// that no row reaches is worth its wait.
constexpr int kResident = 1024;

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
  int32_t rows, nodes, vocab, wide_tokens;
  int32_t pieces, groups;  // of a token's logits; workgroups that take them
  int32_t look;            // whether to look for tokens out of reach
  // between launches 0: what became of each token (see verdict), and who has arrived
  unsigned long long* verdicts;  // [rows][nodes]
  int32_t *node_arrivals, *row_arrivals;
  // not cleared
  struct piece_sum* sums;   // [rows][nodes][pieces]
  struct node_sum* totals;  // [rows][nodes]
  double* rests;            // [rows][pieces]
};

// A piece's largest logit, the first place of it, and the sum of weights beside it
// (NaN: no distribution).
struct piece_sum {
  double z;
  float top;
  int32_t best;
};
struct node_sum {
  double z;
  float top;
  int32_t pad;
};

// Where a row goes from a token: to a child (its number + 2 in the upper half) or nowhere (1);
// 0 is not known yet.  In the lower half the token that follows where it stops.
__device__ __forceinline__ unsigned long long verdict(int child, int token) {
  return (unsigned long long)(uint32_t)(child + 2) << 32 | (uint32_t)token;
}
constexpr int kDraw = -2;  // the token is to be drawn

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


template <typename V>
__device__ __forceinline__ V wave_max(V x) {
  for (int d = 1; d < 64; d *= 2) x = max(x, __shfl_xor(x, d));
  return x;
}
template <typename V>
__device__ __forceinline__ V wave_min(V x) {
  for (int d = 1; d < 64; d *= 2) x = min(x, __shfl_xor(x, d));
  return x;
}
__device__ __forceinline__ double wave_sum(double x) {
  for (int d = 1; d < 64; d *= 2) x += __shfl_xor(x, d);
  return x;
}
struct block_store {
  double d[kWaves];
  int i[kWaves];
  float f[kWaves];
};
__device__ __forceinline__ int block_min(int x, block_store& s) {
  x = wave_min(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s.i[threadIdx.x >> 6] = x;
  __syncthreads();
  return min(min(s.i[0], s.i[1]), min(s.i[2], s.i[3]));
}
__device__ __forceinline__ float block_max(float x, block_store& s) {
  x = wave_max(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s.f[threadIdx.x >> 6] = x;
  __syncthreads();
  return fmaxf(fmaxf(s.f[0], s.f[1]), fmaxf(s.f[2], s.f[3]));
}
// The sum of all threads' numbers before this thread's, and of all.
__device__ __forceinline__ double block_before(double x, double& total, block_store& s) {
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  double run = x;
  for (int d = 1; d < 64; d *= 2) {
    const double lower = __shfl_up(run, d);
    run += lane >= d ? lower : 0.0;
  }
  __syncthreads();
  if (lane == 63) s.d[wave] = run;
  __syncthreads();
  double before = run - x;  // (exact enough: see draw_place)
  total = 0.0;
  for (int w = 0; w < kWaves; ++w) {
    before += w < wave ? s.d[w] : 0.0;
    total += s.d[w];
  }
  return before;
}

// The first place in [0, n) whose running sum, from `before` on, passes `target`: weights
// by `weight_of`, 1024 places at a time.  Where rounding leaves none, the last place of
// any weight (-1: none).
template <typename W>
__device__ __forceinline__ int draw_place(int n, double before, double target, block_store& s, W weight_of) {
  int last = -1;
  for (int v0 = 0; v0 < n; v0 += kThreads * kVec) {
    double w[kVec], mine = 0.0, all;
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      const int v = v0 + (int)threadIdx.x * kVec + e;
      w[e] = v < n ? weight_of(v) : 0.0;
      mine += w[e];
    }
    double upto = before + block_before(mine, all, s);
    int found = INT32_MAX, some = -1;
#pragma unroll
    for (int e = kVec - 1; e >= 0; --e) some = w[e] > 0.0 && some < 0 ? v0 + (int)threadIdx.x * kVec + e : some;
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      upto += w[e];
      if (w[e] > 0.0 && upto > target) found = min(found, v0 + (int)threadIdx.x * kVec + e);
    }
    found = block_min(found, s);
    if (found != INT32_MAX) return found;
    last = max(last, -block_min(-some, s));
    before += all;
  }
  return last;
}

// The piece of `pieces` whose running sum passes `target`, and the sum before it; sums by
// `sum_of`.  (The last piece of any weight where rounding leaves none, -1 where none has.)
template <typename S>
__device__ __forceinline__ int draw_piece(int pieces, double target, double& before, block_store& s, double* s_before,
                                          S sum_of) {
  const int each = (pieces + kThreads - 1) / kThreads, first = (int)threadIdx.x * each;
  double mine = 0.0, total;
  for (int i = first; i < min(first + each, pieces); ++i) mine += sum_of(i);
  double upto = block_before(mine, total, s);
  int found = INT32_MAX, some = -1;
  double found_before = 0.0, some_before = 0.0;
  for (int i = first; i < min(first + each, pieces); ++i) {
    const double w = sum_of(i);
    if (w > 0.0) {
      some = i, some_before = upto;
      if (found == INT32_MAX && upto + w > target) found = i, found_before = upto;
    }
    upto += w;
  }
  int piece = block_min(found, s);
  const bool none = piece == INT32_MAX;
  if (none) piece = -block_min(-some, s);
  if (none ? some == piece && piece >= 0 : found == piece) *s_before = none ? some_before : found_before;
  __syncthreads();
  before = *s_before;
  __syncthreads();
  return piece;
}

template <int DT>
struct row_of {
  typedef typename pl_traits<DT>::T T;
  const verify_args& a;
  const int b, n;
  const float heat;
  const double per;
  __device__ __forceinline__ row_of(const verify_args& args, int row)
      : a(args), b(row), n(args.seq_lens ? min(args.seq_lens[row], args.nodes) : args.nodes),
        heat(args.temperature ? args.temperature[row] : 1.f), per(1.44269504088896340736 / (double)heat) {}
  __device__ __forceinline__ bool greedy() const { return heat == 0.f; }
  __device__ __forceinline__ bool sane() const { return heat >= 0.f && heat < INFINITY; }
  __device__ __forceinline__ const T* logits(int node) const {
    return (const T*)a.logits + b * a.ld_row + node * a.ld_node;
  }
  __device__ __forceinline__ const float* probs(int node) const {
    return a.draft_probs + b * a.ld_draft_row + node * a.ld_draft_node;
  }
  __device__ __forceinline__ int64_t token(int i) const {
    return a.wide_tokens ? ((const int64_t*)a.tokens)[b * a.ld_tokens + i]
                         : ((const int32_t*)a.tokens)[b * a.ld_tokens + i];
  }
  __device__ __forceinline__ int parent(int i) const { return a.parents ? a.parents[b * a.ld_parents + i] : i - 1; }
  __device__ __forceinline__ float uniform_of(int i) const { return a.uniforms[b * a.ld_uniforms + i]; }
};

__device__ __forceinline__ unsigned long long peek(const unsigned long long* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Follows a row's verdicts (all there), writes what comes out and clears them.
template <int DT>
__device__ __forceinline__ void follow(const row_of<DT>& r, int drawn, unsigned long long* s_verdict, int* s_path) {
  const verify_args& a = r.a;
  const int tid = (int)threadIdx.x;
  unsigned long long* verdicts = a.verdicts + (int64_t)r.b * a.nodes;
  __shared__ int s_count, s_token;
  for (int i = tid; i < a.nodes; i += kThreads) {
    s_verdict[i] = peek(verdicts + i);
    s_path[i] = -1;
    __hip_atomic_store(verdicts + i, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (tid == 0) {
    int count = 0, token = -1;
    for (int node = 0; node >= 0 && node < r.n && count < r.n;) {
      s_path[count++] = node;
      const unsigned long long v = s_verdict[node];
      token = (int)(uint32_t)v;
      node = (int)(v >> 32) - 2;
    }
    s_count = count, s_token = token == kDraw ? drawn : token;
  }
  __syncthreads();
  for (int i = tid; i < a.nodes; i += kThreads) a.path[(int64_t)r.b * a.nodes + i] = s_path[i];
  if (tid == 0) a.counts[r.b] = s_count, a.next[r.b] = s_token;
}

// One arrival of a workgroup, behind what it has stored (at agent scope); the count before it.
__device__ __forceinline__ int arrive(int32_t* counter, int add, int* s_old) {
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  __syncthreads();
  if (threadIdx.x == 0)
    *s_old = __hip_atomic_fetch_add(counter, add, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  return *s_old;
}

constexpr int kOut = 1 << 20;  // of an arrival: the token was left out

template <int DT, int PASSES>
__global__ __launch_bounds__(kThreads, 4) void pl_verify_nodes_kernel(verify_args a) {
  typedef typename pl_traits<DT>::T T;
  constexpr int kPiece = 64 * kVec * PASSES;
  __shared__ block_store store;
  __shared__ double s_before;
  __shared__ unsigned long long s_verdict[kNodesMax];
  __shared__ int s_path[kNodesMax];
  __shared__ int s_old;
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int group = (int)(blockIdx.x % a.groups);
  const int b = (int)(blockIdx.x / a.groups % a.rows), node = (int)(blockIdx.x / a.groups / a.rows);
  const row_of<DT> r(a, b);
  unsigned long long* verdicts = a.verdicts + (int64_t)b * a.nodes;
  bool out = node >= r.n;
  if (a.look && node > 0 && !out) {
    // out of reach if a token on the way to it is known to go elsewhere
    for (int i = tid; i <= node; i += kThreads) {
      const int up = i == 0 ? -1 : r.parent(i);
      const unsigned long long v = up >= 0 && up < i ? peek(verdicts + up) : 0;
      // the token before it, or a mark
      s_path[i] = up < 0 || up >= i ? -1 : v && (int)(v >> 32) - 2 != i ? -2 : up;
    }
    __syncthreads();
    int i = node;
    while (i > 0) i = s_path[i];
    out = i == -2;
    __syncthreads();
  }
  piece_sum* sums = a.sums + ((int64_t)b * a.nodes + node) * a.pieces;
  const T* x = r.logits(node);
  if (!out) {
    const int piece = group * kWaves + wave, lo = piece * kPiece, hi = min(lo + kPiece, a.vocab);
    if (piece < a.pieces) {
      float y[PASSES][kVec];
      // rows have the alignment of their elements alone
#pragma unroll
      for (int k = 0; k < PASSES; ++k) {
        const int v = lo + (k * 64 + lane) * kVec;
        if (v + kVec <= hi) {
          T t[kVec];
          __builtin_memcpy(t, x + v, sizeof(t));
#pragma unroll
          for (int e = 0; e < kVec; ++e) y[k][e] = (float)t[e];
        } else {
#pragma unroll
          for (int e = 0; e < kVec; ++e) y[k][e] = v + e < hi ? (float)x[v + e] : -INFINITY;
        }
      }
      float top = -INFINITY;
      bool bad = false;
#pragma unroll
      for (int k = 0; k < PASSES; ++k)
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          bad = bad || !(y[k][e] < INFINITY);
          top = fmaxf(top, y[k][e]);
        }
      bad = __any(bad);
      top = wave_max(top);
      piece_sum sum = {0.0, top, INT32_MAX};
      if (bad || top == -INFINITY) {
        sum.z = bad ? NAN : 0.0;
      } else if (r.greedy()) {
        int best = INT32_MAX;
#pragma unroll
        for (int k = 0; k < PASSES; ++k)
#pragma unroll
          for (int e = 0; e < kVec; ++e)
            if (y[k][e] == top) best = min(best, lo + (k * 64 + lane) * kVec + e);
        sum.best = wave_min(best);
      } else {
        double z = 0.0;
#pragma unroll
        for (int k = 0; k < PASSES; ++k) {
#pragma unroll
          for (int e = 0; e < kVec; ++e) z += weight(y[k][e], top, r.per);
          __builtin_amdgcn_sched_barrier(0);  // a few at a time: other waves fill the gaps
        }
        sum.z = wave_sum(z);
      }
      if (lane == 0) {
        unsigned long long* to = reinterpret_cast<unsigned long long*>(sums + piece);
        __hip_atomic_store(to, __builtin_bit_cast(unsigned long long, sum.z), __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(to + 1, (unsigned long long)(uint32_t)sum.best << 32 | __float_as_uint(sum.top),
                           __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    }
  }
  int32_t* arrivals = a.node_arrivals + (int64_t)b * a.nodes + node;
  const int before = arrive(arrivals, out ? kOut + 1 : 1, &s_old);
  if ((before & (kOut - 1)) != a.groups - 1) return;
  out = out || before >= kOut;
  if (tid == 0) __hip_atomic_store(arrivals, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  // the last of this token: where the row goes from here
  if (!out) {
    auto sum_at = [&](int i) {
      const unsigned long long* from = reinterpret_cast<const unsigned long long*>(sums + i);
      const unsigned long long z = peek(from), rest = peek(from + 1);
      return piece_sum{__builtin_bit_cast(double, z), __uint_as_float((uint32_t)rest), (int)(rest >> 32)};
    };
    float top = -INFINITY;
    bool bad = !r.sane();
    for (int i = tid; i < a.pieces; i += kThreads) {
      const piece_sum p = sum_at(i);
      top = fmaxf(top, p.top), bad = bad || p.z != p.z;
    }
    top = block_max(top, store);
    bad = block_min(bad ? 0 : 1, store) == 0 || top == -INFINITY;
    int child = -1, token = -1;
    if (!bad) {
      int best = INT32_MAX;
      for (int i = tid; r.greedy() && i < a.pieces; i += kThreads) {
        const piece_sum p = sum_at(i);
        if (p.top == top) best = min(best, p.best);
      }
      if (r.greedy()) best = block_min(best, store);
      auto scaled = [&](int i) {
        const piece_sum p = sum_at(i);
        return p.top == -INFINITY ? 0.0 : p.z * weight(p.top, top, r.per);
      };
      double z = 0.0;
      if (!r.greedy()) {
        double mine = 0.0;
        for (int i = tid; i < a.pieces; i += kThreads) mine += scaled(i);
        block_before(mine, z, store);
      }
      if (a.draft_probs) {
        token = r.greedy() ? best : kDraw;
        if (node + 1 < r.n) {
          const int64_t d = r.token(node + 1);
          const bool known = d >= 0 && d < a.vocab;
          const bool go = r.greedy() ? d == best
                                     : known && (double)r.uniform_of(node) * (double)r.probs(node)[d] * z <
                                                    weight((float)x[d], top, r.per);
          child = go ? node + 1 : -1;
        }
        if (tid == 0) a.totals[(int64_t)b * a.nodes + node] = node_sum{z, top, 0};
      } else {
        token = best;
        if (!r.greedy()) {
          const double target = (double)r.uniform_of(node) * z;
          double sum_before = 0.0;
          const int piece = draw_piece(a.pieces, target, sum_before, store, &s_before, scaled);
          const int lo = piece * kPiece;
          token = piece < 0 ? -1
                            : lo + draw_place(min(kPiece, a.vocab - lo), sum_before, target, store,
                                              [&](int v) { return weight((float)x[lo + v], top, r.per); });
        }
        int c = INT32_MAX;
        for (int i = node + 1 + tid; i < r.n; i += kThreads)
          if (r.parent(i) == node && r.token(i) == token) c = min(c, i);
        c = block_min(c, store);
        child = c == INT32_MAX ? -1 : c;
      }
    }
    if (tid == 0)
      __hip_atomic_store(verdicts + node, verdict(child, token), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  if (a.draft_probs) return;  // the second launch follows the row
  if (arrive(a.row_arrivals + b, 1, &s_old) != a.nodes - 1) return;
  if (tid == 0) __hip_atomic_store(a.row_arrivals + b, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  follow(r, -1, s_verdict, s_path);
}

// A line's rows: what follows the token where each stops, drawn from max(e - q Z, 0) there.
template <int DT, int PASSES>
__global__ __launch_bounds__(kThreads) void pl_verify_draw_kernel(verify_args a) {
  typedef typename pl_traits<DT>::T T;
  constexpr int kPiece = 64 * kVec * PASSES;
  __shared__ block_store store;
  __shared__ double s_before;
  __shared__ unsigned long long s_verdict[kNodesMax];
  __shared__ int s_path[kNodesMax];
  __shared__ int s_old;
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int group = (int)(blockIdx.x % a.groups), b = (int)(blockIdx.x / a.groups);
  const row_of<DT> r(a, b);
  const unsigned long long* verdicts = a.verdicts + (int64_t)b * a.nodes;
  // the first token that goes nowhere; those before it all go to the next
  int stop = INT32_MAX;
  for (int i = tid; i < r.n; i += kThreads)
    if (verdicts[i] >> 32 == 1) stop = min(stop, i);
  stop = block_min(stop, store);
  const bool draws = stop < r.n && (int)(uint32_t)verdicts[min(stop, a.nodes - 1)] == kDraw;
  __syncthreads();
  int drawn = -1;
  if (draws) {
    const node_sum total = a.totals[(int64_t)b * a.nodes + stop];
    const T* x = r.logits(stop);
    const float* q = stop + 1 < r.n ? r.probs(stop) : nullptr;
    auto rest_of = [&](float y, float qv) {
      const double e = weight(y, total.top, r.per);
      return fmax(e - (double)qv * total.z, 0.0);
    };
    double* rests = a.rests + (int64_t)b * a.pieces;
    const int piece = group * kWaves + wave, lo = piece * kPiece, hi = min(lo + kPiece, a.vocab);
    if (piece < a.pieces) {
      double z = 0.0;
#pragma unroll 4
      for (int k = 0; k < PASSES; ++k) {
        const int v = lo + (k * 64 + lane) * kVec;
        T t[kVec];
        float p[kVec] = {0.f, 0.f, 0.f, 0.f};
        if (v + kVec <= hi) {
          __builtin_memcpy(t, x + v, sizeof(t));
          if (q) __builtin_memcpy(p, q + v, sizeof(p));
#pragma unroll
          for (int e = 0; e < kVec; ++e) z += rest_of((float)t[e], p[e]);
        } else {
          for (int e = 0; v + e < hi; ++e) z += rest_of((float)x[v + e], q ? q[v + e] : 0.f);
        }
      }
      z = wave_sum(z);
      if (lane == 0)
        __hip_atomic_store(reinterpret_cast<unsigned long long*>(rests + piece),
                           __builtin_bit_cast(unsigned long long, z), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if (arrive(a.row_arrivals + b, 1, &s_old) != a.groups - 1) return;
    if (tid == 0) __hip_atomic_store(a.row_arrivals + b, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    auto rest_at = [&](int i) {
      return __builtin_bit_cast(double, peek(reinterpret_cast<const unsigned long long*>(rests + i)));
    };
    const float u = r.uniform_of(r.n - 1);
    double mine = 0.0, all;
    for (int i = tid; i < a.pieces; i += kThreads) mine += rest_at(i);
    block_before(mine, all, store);
    if (q && !(all > 0.0)) {
      // p and q agree everywhere: from p itself
      const piece_sum* sums = a.sums + ((int64_t)b * a.nodes + stop) * a.pieces;
      auto scaled = [&](int i) {
        return sums[i].top == -INFINITY ? 0.0 : sums[i].z * weight(sums[i].top, total.top, r.per);
      };
      const double target = (double)u * total.z;
      double before = 0.0;
      const int at = draw_piece(a.pieces, target, before, store, &s_before, scaled);
      if (at >= 0)
        drawn = at * kPiece + draw_place(min(kPiece, a.vocab - at * kPiece), before, target, store,
                                         [&](int v) { return weight((float)x[at * kPiece + v], total.top, r.per); });
    } else {
      const double target = (double)u * all;
      double before = 0.0;
      const int at = draw_piece(a.pieces, target, before, store, &s_before, rest_at);
      if (at >= 0)
        drawn = at * kPiece + draw_place(min(kPiece, a.vocab - at * kPiece), before, target, store, [&](int v) {
                  return rest_of((float)x[at * kPiece + v], q ? q[at * kPiece + v] : 0.f);
                });
    }
  } else if (group != 0) {
    return;
  }
  follow(r, drawn, s_verdict, s_path);
}

// Rows of no token.
__global__ __launch_bounds__(kThreads) void pl_verify_none_kernel(int32_t* counts, int64_t* next, int32_t rows) {
  const int b = (int)(blockIdx.x * kThreads + threadIdx.x);
  if (b < rows) counts[b] = 0, next[b] = -1;
}

// How a call is cut: pieces of a token's logits, and the workgroups that take them.
struct verify_cut {
  int passes, pieces, groups;
};
verify_cut cut_of(int64_t rows, int64_t nodes, int64_t vocab) {
  verify_cut c;
  const int64_t few = (vocab + 64 * kVec * kFewPasses - 1) / (64 * kVec * kFewPasses);
  c.passes = rows * nodes * few > kManyPieces ? kManyPasses : kFewPasses;
  const int64_t piece = 64 * kVec * c.passes;
  c.pieces = (int)((vocab + piece - 1) / piece);
  c.groups = (c.pieces + kWaves - 1) / kWaves;
  if (c.groups == 0) c.groups = 1;
  return c;
}

template <int DT, int PASSES>
int launch(const verify_args& a, hipStream_t s) {
  const char* what = "pl_verify_tokens";
  pl_verify_nodes_kernel<DT, PASSES><<<dim3((unsigned)(a.rows * a.nodes * a.groups)), kThreads, 0, s>>>(a);
  const int rc = pl_launch_status(what);
  if (rc || !a.draft_probs) return rc;
  pl_verify_draw_kernel<DT, PASSES><<<dim3((unsigned)(a.rows * a.groups)), kThreads, 0, s>>>(a);
  return pl_launch_status(what);
}
template <int DT>
int launch(const verify_args& a, int passes, hipStream_t s) {
  return passes == kFewPasses ? launch<DT, kFewPasses>(a, s) : launch<DT, kManyPasses>(a, s);
}

int64_t whole_pieces(int64_t bytes) { return (bytes + 255) / 256 * 256; }

}  // namespace

extern "C" int64_t pl_verify_workspace_bytes(int32_t rows, int32_t nodes, int32_t vocab) {
  if (rows < 0 || nodes < 0 || vocab < 0) return 0;
  const verify_cut c = cut_of(rows, nodes, vocab);
  const int64_t n = (int64_t)rows * nodes;
  return whole_pieces(n * c.pieces * (int64_t)sizeof(piece_sum)) + whole_pieces(n * (int64_t)sizeof(node_sum)) +
         whole_pieces((int64_t)rows * c.pieces * 8);
}
extern "C" int64_t pl_verify_counter_ints(int32_t rows, int32_t nodes) {
  return rows < 0 || nodes < 0 ? 0 : 3ll * rows * nodes + rows;
}

extern "C" int pl_verify_tokens(int32_t dtype, const void* logits, int64_t ld_row, int64_t ld_node,
                                const void* tokens, int32_t token_bytes, int64_t ld_tokens,
                                const float* uniforms, int64_t ld_uniforms, const int32_t* parents,
                                int64_t ld_parents, const float* draft_probs, int64_t ld_draft_row,
                                int64_t ld_draft_node, const float* temperature, const int32_t* seq_lens,
                                int32_t rows, int32_t nodes, int32_t vocab, int32_t* path, int32_t* counts,
                                int64_t* next, void* workspace, int64_t workspace_bytes, int32_t* counters,
                                int64_t counter_ints, void* stream) {
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
  if (vocab > kVocabMax || nodes > kNodesMax) {
    pl_set_error("%s: at most %d logits to a token and %d tokens to a row (got %d and %d)", what, kVocabMax, kNodesMax,
                 vocab, nodes);
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
  const int64_t need = pl_verify_workspace_bytes(rows, nodes, vocab), ints = pl_verify_counter_ints(rows, nodes);
  if (!workspace || workspace_bytes < need || !counters || counter_ints < ints) {
    pl_set_error("%s: workspace of %lld bytes and %lld counters, %lld and %lld needed", what,
                 (long long)workspace_bytes, (long long)counter_ints, (long long)need, (long long)ints);
    return PL_ERR_ARG;
  }
  verify_args a;
  a.logits = logits, a.ld_row = ld_row, a.ld_node = ld_node, a.tokens = tokens, a.ld_tokens = ld_tokens;
  a.uniforms = uniforms, a.ld_uniforms = ld_uniforms, a.parents = parents, a.ld_parents = ld_parents;
  a.draft_probs = draft_probs, a.ld_draft_row = ld_draft_row, a.ld_draft_node = ld_draft_node;
  a.temperature = temperature, a.seq_lens = seq_lens, a.path = path, a.counts = counts, a.next = next;
  a.rows = rows, a.nodes = nodes, a.vocab = vocab, a.wide_tokens = token_bytes == 8;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (nodes == 0) {
    pl_verify_none_kernel<<<dim3((unsigned)((rows + kThreads - 1) / kThreads)), kThreads, 0, s>>>(counts, next, rows);
    return pl_launch_status(what);
  }
  const verify_cut c = cut_of(rows, nodes, vocab);
  a.pieces = c.pieces, a.groups = c.groups;
  const int64_t blocks = (int64_t)rows * nodes * c.groups, n = (int64_t)rows * nodes;
  if (!pl_grid_fits(blocks, kThreads) || blocks > INT32_MAX) {
    pl_set_error("%s: too many rows (%d)", what, rows);
    return PL_ERR_LIMIT;
  }
  a.look = blocks > kResident;
  uint8_t* at = static_cast<uint8_t*>(workspace);
  a.sums = reinterpret_cast<piece_sum*>(at), at += whole_pieces(n * c.pieces * (int64_t)sizeof(piece_sum));
  a.totals = reinterpret_cast<node_sum*>(at), at += whole_pieces(n * (int64_t)sizeof(node_sum));
  a.rests = reinterpret_cast<double*>(at);
  a.verdicts = reinterpret_cast<unsigned long long*>(counters);
  a.node_arrivals = counters + 2 * n, a.row_arrivals = counters + 3 * n;
  if (dtype == PL_F32) return launch<PL_F32>(a, c.passes, s);
  return dtype == PL_BF16 ? launch<PL_BF16>(a, c.passes, s) : launch<PL_F16>(a, c.passes, s);
}
