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
// A launch looks at all tokens of all rows at once, a wave to a piece of a token's
// logits, which it reads once into registers: the largest, then the sum of weights
// beside that.  Few tokens are spread over workgroups of four pieces, and a second
// launch, a workgroup to a token, puts their sums together and says where the row would
// go from there; of many, each has a workgroup that does both.  A last launch follows
// each row.  Many tokens' workgroups do not run all at once: tokens lie in the grid's
// order before those behind them, and a workgroup leaves out a token
// that a row is known to have turned away from: what it would have found counts
// for nothing.  Drawing from what is left of p beside q needs Z first: its pieces are a
// launch of their own, before the last.
//
// What a workgroup finds goes to others from launch to launch only.  Handing it on inside of
// one takes a release and an acquire at agent scope, 22 to 33 ns of the whole GPU's time for every
// workgroup that has something (256 rows: 1786 us), and without them nothing promises
// that who arrives last at a counter sees what the others have stored: neighbouring tokens' sums
// share lines, which an XCD that has read one token's may still hold when it reads the next one's.
//
// 64-bit exponentials bound a batch: 256 rows of 6 tokens over 128256 fp32 logits take 170 to 190 us, 89
// of them their bytes at a copy's rate; without the exponentials the time was nearly halved.
// One row takes 19 us, four launches that each wait for a few reads one after the other.
// A workgroup that draws a row whole, without a launch for its pieces, was faster at no
// number of rows (256 rows of 2 tokens over 128256 fp32 logits 93 and 93 us, 64 rows 57 and 36, 1024 rows
// over 32003 118 and 99).
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kVec = 4, kPasses = 4;  // logits of a lane's load, and its loads to a piece
constexpr int kPiece = 64 * kVec * kPasses;
constexpr int kNodesMax = 1024;  // tokens of a row
constexpr int kVocabMax = 1 << 24;
// Threads of a workgroup that takes a token whole, and tokens of a call above which there
// are such.  Pieces in workgroups of four spread a call over the GPU at once; where that
// has many to follow one another, a token's workgroup pays what one costs besides
// its logits once, and of the tokens behind others only a few begin before those are
// done.  Measured in us, whole and spread: 32 tokens a row of 32003 bf16, 512 tokens 33 and 29, 2048
// 77 and 68, 4096 103 and 124; 6 a row of 128256 in fp32, 384 tokens 79 and 60, 768 123 and 107, 1536 194
// and 197.
constexpr int kWholeThreads = 1024;
constexpr int kWholeTokens = 1024, kWholeFewTokens = 2048;
constexpr int kFewPieces = 64;  // up to these such a workgroup has kThreads: less to wait for
constexpr int kWholePieces = 1024;  // whose sums fit beside it

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
  unsigned long long* verdicts;  // [rows][nodes]: what became of each token (see verdict); between calls 0
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

// 2^t, |t| up to 1000, to 2e-14 of it: the power of two of the nearest integer, which the
// sum with 1.5 * 2^52 holds in its lowest bits and adds to the exponent, times the
// Chebyshev interpolation of degree 9 of 2^f for the rest, f in [-1/2, 1/2] (computed
// from its definition in 60 digits).
__device__ __forceinline__ double exp2_64(double t) {
  constexpr double kRound = 6755399441055744.0;
  const double n = t + kRound, f = t - (n - kRound);
  double p = 0x1.b6571de2f2351p-24;
  p = fma(p, f, 0x1.63ef969a64d3cp-20);
  p = fma(p, f, 0x1.ffcb76789860fp-17);
  p = fma(p, f, 0x1.43088e257f341p-13);
  p = fma(p, f, 0x1.5d87fe908f88ap-10);
  p = fma(p, f, 0x1.3b2ab72b175eep-7);
  p = fma(p, f, 0x1.c6b08d7044119p-5);
  p = fma(p, f, 0x1.ebfbdff8149f2p-3);
  p = fma(p, f, 0x1.62e42fefa39f7p-1);
  p = fma(p, f, 0x1.000000000003dp+0);
  const uint64_t bits = __builtin_bit_cast(uint64_t, p);
  const uint32_t high = (uint32_t)(bits >> 32) + ((uint32_t)__builtin_bit_cast(uint64_t, n) << 20);
  return __builtin_bit_cast(double, (uint64_t)high << 32 | (uint32_t)bits);
}

// The weight of a logit (no NaN) beside a reference, `per` = log2(e) / temperature; never less
// than 2^-1000, what -infinity gives.
__device__ __forceinline__ double weight_least(float x, float top, double per) {
  return exp2_64(fmax(((double)x - (double)top) * per, -1000.0));
}
// And with 0 for -infinity.
__device__ __forceinline__ double weight(float x, float top, double per) {
  return x == -INFINITY ? 0.0 : weight_least(x, top, per);
}
// A piece's sum of weights without what those put in that stand for 0 (the choice in each of them took a
// tenth of a large batch's time).
__device__ __forceinline__ double without_least(double z) { return z < 0x1p-900 ? 0.0 : z; }

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
// The sum of a wave's numbers, in lane 63: shifts by 1, 2, 4 and 8 inside rows of 16, then each
// row's last lane into the rows above.
template <int CTRL, int ROWS>
__device__ __forceinline__ double from_lower(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, ROWS, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, ROWS, 0xf, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double wave_sum(double x) {
  x += from_lower<0x111, 0xf>(x), x += from_lower<0x112, 0xf>(x);
  x += from_lower<0x114, 0xf>(x), x += from_lower<0x118, 0xf>(x);
  x += from_lower<0x142, 0xa>(x);
  return x + from_lower<0x143, 0xc>(x);
}
template <int THREADS>
struct block_store {
  double d[THREADS / 64];
  int i[THREADS / 64];
  float f[THREADS / 64];
};
template <int THREADS>
__device__ __forceinline__ int block_min(int x, block_store<THREADS>& s) {
  x = wave_min(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s.i[threadIdx.x >> 6] = x;
  __syncthreads();
  x = s.i[0];
#pragma unroll
  for (int w = 1; w < THREADS / 64; ++w) x = min(x, s.i[w]);
  return x;
}
template <int THREADS>
__device__ __forceinline__ float block_max(float x, block_store<THREADS>& s) {
  x = wave_max(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s.f[threadIdx.x >> 6] = x;
  __syncthreads();
  x = s.f[0];
#pragma unroll
  for (int w = 1; w < THREADS / 64; ++w) x = fmaxf(x, s.f[w]);
  return x;
}
// The sum of all threads' numbers before this thread's, and of all.
template <int THREADS>
__device__ __forceinline__ double block_before(double x, double& total, block_store<THREADS>& s) {
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
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    before += w < wave ? s.d[w] : 0.0;
    total += s.d[w];
  }
  return before;
}

// The first place in [0, n) whose running sum, from `before` on, passes `target`: weights
// by `weight_of`, four places of a thread at a time.  Where rounding leaves none, the last place of
// any weight (-1: none).
template <int THREADS, typename W>
__device__ __forceinline__ int draw_place(int n, double before, double target, block_store<THREADS>& s, W weight_of) {
  int last = -1;
  for (int v0 = 0; v0 < n; v0 += THREADS * kVec) {
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
template <int THREADS, typename S>
__device__ __forceinline__ int draw_piece(int pieces, double target, double& before, block_store<THREADS>& s,
                                          double* s_before, S sum_of) {
  const int each = (pieces + THREADS - 1) / THREADS, first = (int)threadIdx.x * each;
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

// Whether a token is out of a row's reach: a token on the way to it is known to go elsewhere.
template <int THREADS, int DT>
__device__ __forceinline__ bool out_of_reach(const row_of<DT>& r, int node, const unsigned long long* verdicts,
                                             int* s_path) {
  for (int i = (int)threadIdx.x; i <= node; i += THREADS) {
    const int up = i == 0 ? -1 : r.parent(i);
    const unsigned long long v = up >= 0 && up < i ? peek(verdicts + up) : 0;
    // the token before it, or a mark
    s_path[i] = up < 0 || up >= i ? -1 : v && (int)(v >> 32) - 2 != i ? -2 : up;
  }
  __syncthreads();
  int i = node;
  while (i > 0) i = s_path[i];
  __syncthreads();
  return i == -2;
}

// A piece of a row's logits in registers; `none` past their end.
template <typename T>
__device__ __forceinline__ void load_piece(const T* x, int lo, int vocab, float (&y)[kPasses][kVec], float none) {
  const int lane = (int)threadIdx.x & 63;
  // rows have the alignment of their elements alone
#pragma unroll
  for (int k = 0; k < kPasses; ++k) {
    const int v = lo + (k * 64 + lane) * kVec;
    if (v + kVec <= vocab) {
      T t[kVec];
      __builtin_memcpy(t, x + v, sizeof(t));
#pragma unroll
      for (int e = 0; e < kVec; ++e) y[k][e] = (float)t[e];
    } else {
#pragma unroll
      for (int e = 0; e < kVec; ++e) y[k][e] = v + e < vocab ? (float)x[v + e] : none;
    }
  }
}

// A piece's sum (in lane 63) beside `ref`, which rises to its largest logit where that is none yet, or
// so far above that weights would leave 64 bits (2^500).
template <int DT>
__device__ __forceinline__ piece_sum sum_piece(const row_of<DT>& r, const float (&y)[kPasses][kVec], int lo, float& ref) {
  const int lane = (int)threadIdx.x & 63;
  float top = -INFINITY;
  bool bad = false;
#pragma unroll
  for (int k = 0; k < kPasses; ++k)
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      bad = bad || !(y[k][e] < INFINITY);
      top = fmaxf(top, y[k][e]);
    }
  if (__any(bad)) return {NAN, top, INT32_MAX};
  if (r.greedy()) {
    top = wave_max(top);
    int best = INT32_MAX;
#pragma unroll
    for (int k = 0; k < kPasses; ++k)
#pragma unroll
      for (int e = 0; e < kVec; ++e)
        if (y[k][e] == top) best = min(best, lo + (k * 64 + lane) * kVec + e);
    return {0.0, top, wave_min(best)};
  }
  if (__any(ref == -INFINITY || ((double)top - (double)ref) * r.per > 500.0)) ref = wave_max(top);
  if (ref == -INFINITY) return {0.0, ref, INT32_MAX};
  double z = 0.0;
#pragma unroll
  for (int k = 0; k < kPasses; ++k) {
#pragma unroll
    for (int e = 0; e < kVec; ++e) z += weight_least(y[k][e], ref, r.per);
    __builtin_amdgcn_sched_barrier(0);  // a few at a time: other waves fill the gaps
  }
  return {without_least(wave_sum(z)), ref, INT32_MAX};
}

// Where the row goes from a token, from its pieces' sums.
template <int THREADS, int DT, typename S>
__device__ __forceinline__ unsigned long long resolve(const row_of<DT>& r, int node, S sum_at,
                                                      block_store<THREADS>& store, double* s_before) {
  const verify_args& a = r.a;
  const int tid = (int)threadIdx.x;
  const auto* x = r.logits(node);
  float top = -INFINITY;
  bool bad = !r.sane();
  for (int i = tid; i < a.pieces; i += THREADS) {
    const piece_sum p = sum_at(i);
    top = fmaxf(top, p.top), bad = bad || p.z != p.z;
  }
  top = block_max(top, store);
  bad = block_min(bad ? 0 : 1, store) == 0 || top == -INFINITY;
  if (bad) return verdict(-1, -1);
  int child = -1, token = -1, best = INT32_MAX;
  if (r.greedy()) {
    for (int i = tid; i < a.pieces; i += THREADS) {
      const piece_sum p = sum_at(i);
      if (p.top == top) best = min(best, p.best);
    }
    best = block_min(best, store);
  }
  auto scaled = [&](int i) {
    const piece_sum p = sum_at(i);
    return p.top == -INFINITY ? 0.0 : p.z * weight(p.top, top, r.per);
  };
  double z = 0.0;
  if (!r.greedy()) {
    double mine = 0.0;
    for (int i = tid; i < a.pieces; i += THREADS) mine += scaled(i);
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
    if (tid == 0) a.totals[(int64_t)r.b * a.nodes + node] = node_sum{z, top, 0};
  } else {
    token = best;
    if (!r.greedy()) {
      const double target = (double)r.uniform_of(node) * z;
      double before = 0.0;
      const int piece = draw_piece(a.pieces, target, before, store, s_before, scaled), lo = piece * kPiece;
      token = piece < 0 ? -1
                        : lo + draw_place(min(kPiece, a.vocab - lo), before, target, store,
                                          [&](int v) { return weight((float)x[lo + v], top, r.per); });
    }
    int c = INT32_MAX;
    for (int i = node + 1 + tid; i < r.n; i += THREADS)
      if (r.parent(i) == node && r.token(i) == token) c = min(c, i);
    c = block_min(c, store);
    child = c == INT32_MAX ? -1 : c;
  }
  return verdict(child, token);
}

// A wave to each piece of a token.
template <int DT>
__global__ __launch_bounds__(kThreads) void pl_verify_pieces_kernel(verify_args a) {
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  const int group = (int)(blockIdx.x % a.groups);
  const int b = (int)(blockIdx.x / a.groups % a.rows), node = (int)(blockIdx.x / a.groups / a.rows);
  const row_of<DT> r(a, b);
  const int piece = group * kWaves + wave;
  if (node >= r.n || piece >= a.pieces) return;
  float y[kPasses][kVec], ref = -INFINITY;
  load_piece(r.logits(node), piece * kPiece, a.vocab, y, -INFINITY);
  const piece_sum sum = sum_piece(r, y, piece * kPiece, ref);
  if (lane == 63) a.sums[((int64_t)b * a.nodes + node) * a.pieces + piece] = sum;
}

// And a workgroup to each token, for what its pieces say.
template <int DT>
__global__ __launch_bounds__(kThreads) void pl_verify_resolve_kernel(verify_args a) {
  __shared__ block_store<kThreads> store;
  __shared__ double s_before;
  const int b = (int)(blockIdx.x % a.rows), node = (int)(blockIdx.x / a.rows);
  const row_of<DT> r(a, b);
  if (node >= r.n) return;
  const int64_t at = (int64_t)b * a.nodes + node;
  const piece_sum* sums = a.sums + at * a.pieces;
  const unsigned long long v = resolve(r, node, [&](int i) { return sums[i]; }, store, &s_before);
  if (threadIdx.x == 0) a.verdicts[at] = v;
}

// A workgroup to each token, its waves taking pieces in turn.
template <int DT, int THREADS>
__global__ __launch_bounds__(THREADS, 8) void pl_verify_whole_kernel(verify_args a) {
  __shared__ block_store<THREADS> store;
  __shared__ double s_before;
  __shared__ piece_sum s_sums[THREADS == kThreads ? kFewPieces : kWholePieces];
  __shared__ int s_path[kNodesMax];
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int b = (int)(blockIdx.x % a.rows), node = (int)(blockIdx.x / a.rows);
  const row_of<DT> r(a, b);
  unsigned long long* verdicts = a.verdicts + (int64_t)b * a.nodes;
  if (node >= r.n) return;
  if (node > 0 && out_of_reach<THREADS>(r, node, verdicts, s_path)) return;
  constexpr int kStep = THREADS / 64;
  float y[kPasses][kVec], ref = -INFINITY;
  for (int piece = wave; piece < a.pieces; piece += kStep) {
    load_piece(r.logits(node), piece * kPiece, a.vocab, y, -INFINITY);
    const piece_sum sum = sum_piece(r, y, piece * kPiece, ref);
    if (lane == 63) s_sums[piece] = sum;
  }
  __syncthreads();
  const unsigned long long v = resolve(r, node, [&](int i) { return s_sums[i]; }, store, &s_before);
  // what a draw may ask for once more
  if (a.draft_probs)
    for (int i = tid; i < a.pieces; i += THREADS)
      a.sums[((int64_t)b * a.nodes + node) * a.pieces + i] = s_sums[i];
  if (tid == 0) __hip_atomic_store(verdicts + node, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// What a row of a line draws from, max(e - q Z, 0) at the token where it stops (verdicts all there).
template <int DT>
struct rest_of {
  typedef typename pl_traits<DT>::T T;
  const row_of<DT>& r;
  int stop;
  bool draws;  // the row stops, and at usable logits
  node_sum total;
  const T* x;
  const float* q;  // null behind the last draft
  __device__ __forceinline__ rest_of(const row_of<DT>& row, block_store<kThreads>& store) : r(row) {
    const verify_args& a = r.a;
    const unsigned long long* verdicts = a.verdicts + (int64_t)r.b * a.nodes;
    // the first token that goes nowhere; those before it all go to the next
    stop = INT32_MAX;
    for (int i = (int)threadIdx.x; i < r.n; i += kThreads)
      if (verdicts[i] >> 32 == 1) stop = min(stop, i);
    stop = block_min(stop, store);
    draws = stop < r.n && (int)(uint32_t)verdicts[min(stop, a.nodes - 1)] == kDraw;
    __syncthreads();
    total = draws ? a.totals[(int64_t)r.b * a.nodes + stop] : node_sum{0.0, 0.f, 0};
    x = r.logits(draws ? stop : 0);
    q = draws && stop + 1 < r.n ? r.probs(stop) : nullptr;
  }
  __device__ __forceinline__ double of(double e, float qv) const { return fmax(e - (double)qv * total.z, 0.0); }
  // A piece's sum of them, in lane 63.
  __device__ __forceinline__ double piece(int i) const {
    float y[kPasses][kVec], p[kPasses][kVec] = {};
    load_piece(x, i * kPiece, r.a.vocab, y, -INFINITY);
    if (q) load_piece(q, i * kPiece, r.a.vocab, p, 0.f);
    double z = 0.0;
#pragma unroll
    for (int k = 0; k < kPasses; ++k) {
#pragma unroll
      for (int e = 0; e < kVec; ++e) z += of(weight_least(y[k][e], total.top, r.per), p[k][e]);
      __builtin_amdgcn_sched_barrier(0);
    }
    return without_least(wave_sum(z));
  }
};

// The pieces' sums of that, a wave to each.
template <int DT>
__global__ __launch_bounds__(kThreads) void pl_verify_rests_kernel(verify_args a) {
  __shared__ block_store<kThreads> store;
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  const int group = (int)(blockIdx.x % a.groups), b = (int)(blockIdx.x / a.groups);
  const row_of<DT> r(a, b);
  const rest_of<DT> rest(r, store);
  const int i = group * kWaves + wave;
  if (!rest.draws || i >= a.pieces) return;
  const double z = rest.piece(i);
  if (lane == 63) a.rests[(int64_t)b * a.pieces + i] = z;
}

// Follows each row.  Of lines it draws what follows the token where each stops, from the pieces' sums.
template <int DT>
__global__ __launch_bounds__(kThreads) void pl_verify_follow_kernel(verify_args a) {
  __shared__ block_store<kThreads> store;
  __shared__ double s_before;
  __shared__ unsigned long long s_verdict[kNodesMax];
  __shared__ int s_path[kNodesMax];
  __shared__ int s_count, s_token;
  const int tid = (int)threadIdx.x, b = (int)blockIdx.x;
  const row_of<DT> r(a, b);
  unsigned long long* verdicts = a.verdicts + (int64_t)b * a.nodes;
  int drawn = -1;
  if (a.draft_probs) {
    rest_of<DT> rest(r, store);
    if (rest.draws) {
      const double* rests = a.rests + (int64_t)b * a.pieces;
      const float u = r.uniform_of(r.n - 1);
      double mine = 0.0, all, before = 0.0;
      for (int i = tid; i < a.pieces; i += kThreads) mine += rests[i];
      block_before(mine, all, store);
      // where p and q agree everywhere, from p itself
      const bool whole = rest.q && !(all > 0.0);
      if (whole) rest.q = nullptr, all = rest.total.z;
      const double target = (double)u * all;
      const piece_sum* sums = a.sums + ((int64_t)b * a.nodes + rest.stop) * a.pieces;
      const int at = draw_piece(a.pieces, target, before, store, &s_before, [&](int i) {
        if (!whole) return rests[i];
        return sums[i].top == -INFINITY ? 0.0 : sums[i].z * weight(sums[i].top, rest.total.top, r.per);
      });
      if (at >= 0) {
        const int lo = at * kPiece;
        drawn = lo + draw_place(min(kPiece, a.vocab - lo), before, target, store, [&](int v) {
                  return rest.of(weight((float)rest.x[lo + v], rest.total.top, r.per), rest.q ? rest.q[lo + v] : 0.f);
                });
      }
    }
  }
  for (int i = tid; i < a.nodes; i += kThreads) {
    s_verdict[i] = verdicts[i];
    s_path[i] = -1;
    verdicts[i] = 0;  // as the next call expects them
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
  for (int i = tid; i < a.nodes; i += kThreads) a.path[(int64_t)b * a.nodes + i] = s_path[i];
  if (tid == 0) a.counts[b] = s_count, a.next[b] = s_token;
}

// Rows of no token.
__global__ __launch_bounds__(kThreads) void pl_verify_none_kernel(int32_t* counts, int64_t* next, int32_t rows) {
  const int b = (int)(blockIdx.x * kThreads + threadIdx.x);
  if (b < rows) counts[b] = 0, next[b] = -1;
}

int pieces_of(int64_t vocab) { return (int)((vocab + kPiece - 1) / kPiece); }

template <int DT>
int launch(const verify_args& a, bool whole, hipStream_t s) {
  const char* what = "pl_verify_tokens";
  const dim3 tokens((unsigned)a.rows * (unsigned)a.nodes), rows((unsigned)a.rows);
  int rc;
  if (whole && a.pieces <= kFewPieces) {
    pl_verify_whole_kernel<DT, kThreads><<<tokens, kThreads, 0, s>>>(a);
  } else if (whole) {
    pl_verify_whole_kernel<DT, kWholeThreads><<<tokens, kWholeThreads, 0, s>>>(a);
  } else {
    pl_verify_pieces_kernel<DT><<<dim3(tokens.x * (unsigned)a.groups), kThreads, 0, s>>>(a);
    if ((rc = pl_launch_status(what))) return rc;
    pl_verify_resolve_kernel<DT><<<tokens, kThreads, 0, s>>>(a);
  }
  if ((rc = pl_launch_status(what))) return rc;
  if (a.draft_probs) {
    pl_verify_rests_kernel<DT><<<dim3(rows.x * (unsigned)a.groups), kThreads, 0, s>>>(a);
    if ((rc = pl_launch_status(what))) return rc;
  }
  pl_verify_follow_kernel<DT><<<rows, kThreads, 0, s>>>(a);
  return pl_launch_status(what);
}

int64_t whole_pieces(int64_t bytes) { return (bytes + 255) / 256 * 256; }

}  // namespace

extern "C" int64_t pl_verify_workspace_bytes(int32_t rows, int32_t nodes, int32_t vocab) {
  if (rows < 0 || nodes < 0 || vocab < 0) return 0;
  const int64_t n = (int64_t)rows * nodes, pieces = pieces_of(vocab);
  return whole_pieces(n * pieces * (int64_t)sizeof(piece_sum)) + whole_pieces(n * (int64_t)sizeof(node_sum)) +
         whole_pieces((int64_t)rows * pieces * 8);
}
extern "C" int64_t pl_verify_counter_ints(int32_t rows, int32_t nodes) {
  return rows < 0 || nodes < 0 ? 0 : 2ll * rows * nodes;
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
  if (reinterpret_cast<uintptr_t>(workspace) % 128 != 0 || reinterpret_cast<uintptr_t>(counters) % 8 != 0) {
    pl_set_error("%s: the workspace must begin at whole 128 bytes, the counters at whole 8", what);
    return PL_ERR_ALIGN;
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
  const int64_t n = (int64_t)rows * nodes;
  a.pieces = pieces_of(vocab), a.groups = a.pieces > kWaves ? (a.pieces + kWaves - 1) / kWaves : 1;
  const bool few = a.pieces <= kFewPieces;
  const bool whole = n > (few ? kWholeFewTokens : kWholeTokens) && a.pieces <= kWholePieces;
  // the first launch's workgroups, and the pieces' of a draw
  if (!(whole ? pl_grid_fits(n, few ? kThreads : kWholeThreads) : pl_grid_fits(n * a.groups, kThreads)) ||
      !pl_grid_fits(draft_probs ? (int64_t)rows * a.groups : rows, kThreads)) {
    pl_set_error("%s: too many rows (%d)", what, rows);
    return PL_ERR_LIMIT;
  }
  uint8_t* at = static_cast<uint8_t*>(workspace);
  a.sums = reinterpret_cast<piece_sum*>(at), at += whole_pieces(n * a.pieces * (int64_t)sizeof(piece_sum));
  a.totals = reinterpret_cast<node_sum*>(at), at += whole_pieces(n * (int64_t)sizeof(node_sum));
  a.rests = reinterpret_cast<double*>(at);
  a.verdicts = reinterpret_cast<unsigned long long*>(counters);
  if (dtype == PL_F32) return launch<PL_F32>(a, whole, s);
  return dtype == PL_BF16 ? launch<PL_BF16>(a, whole, s) : launch<PL_F16>(a, whole, s);
}
