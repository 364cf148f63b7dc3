// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
// The walk over a sequence's tree (draft.h) starts at node 0. At a node, r = p = softmax(logits /
// temperature) of its row; its children x, in order, are tested one after another:
//   accepted when u_x q(x) < r(x)          (u_x the child's uniform number): the walk goes on there
//   else r <- max(r - q, 0), normalised    (a sum of 0 leaves r as it is)
// q is the drafter's distribution of the node's children (draft_probs row of the node), or, when the
// drafts were given without probabilities, 1 at the child's token. When no child is accepted, the
// next token is argmax r(v) / E(v) with the sequence's Exp(1) noise (the exponential race of
// sampling.hip). A temperature below 1e-5 takes the child whose token is the row's argmax, and the
// argmax at the end. Accepting and sampling this way leaves every token distributed as p.
//
// The emitted tokens are thus the drafts on the accepted path and one more. A row whose softmax is not
// a number accepts nothing and gives token 0, as the sampler does; tokens of probability 0 are never given.
//
// r after k rejections is (p - c_k q)+ / N_k, with c_0 = 0, N_0 = 1, c_{k+1} = c_k + N_k and
// N_k = sum (p - c_k q)+, since ((p - c q)+ / N - q)+ = (p - (c + N) q)+ / N: one number stands for a chain
// of rejections. With given drafts it is p with the rejected tokens struck out, over what is left of 1.
//
// Four launches, or three: small batches walk inside the race. The softmax (greedy: the argmax) of rows that have children, cut into slices that
// all CUs share; the walks, a lane for each node, every lane with its own test's numbers in registers; the
// race for the last token over slices of the last row, as maxima of (key, index) words; their maximum. (A
// last slice that joins them, by an atomic count, took longer: what the other XCDs wrote has to be made
// visible to it, 9.7 us against 4 and a launch for one stream.) The race compares log2(e) (x - m) / temperature - log2 E, m
// the largest x of a wavefront's part and then of a slice, taken along and made up for where parts are joined: it needs no
// softmax, and sees no shift of a row, as a softmax does not (without m, logits of 10^4 at temperature 0.01
// had keys of 10^6, and the noise was rounded off).
//
// Many rows (large trees) would be read for nothing: a walk visits a few of a tree's rows. There, the first
// launch is one for each of the path's first kLevels nodes: every workgroup takes the step from the node
// before, from its slices, and reads a slice of the node it comes to. Deeper nodes, and drawn drafts, whose
// residuals are sums over rows, are left to the walk, whose workgroup reads each row when it gets there.
// 24 trees of up to 64 nodes with 152K tokens, paths of up to 6: a launch takes
// 6 us, 61 to 71 us in all; with every row read by the walk's own workgroup (12 us a row, its CU's exponentials) it was 89.
// One stream of 5 nodes: 15.5 us, three launches from the host; 32 chains with their drafter's distributions: 41 us, 2.1 TB/s
// (rows 16, walks 10, race 14).
#include <algorithm>

#include "draft.h"

namespace {

using lsh::DraftSeq;
using lsh::kWave;
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));  // (rows of an odd vocabulary)

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kSliceThreads = 256;      // the workgroup of a slice of a row
constexpr int kPer = 4;                 // its 16-byte loads for each thread
constexpr int kSlice = kSliceThreads * kPer * 4;  // tokens of a slice
constexpr int kWalkWaves = 16;          // of the workgroup of a walk that reads rows itself
// Logits up to which the rows' softmaxes are formed ahead of the walks: of drawn drafts, and of given ones (trees of up to
// 58 nodes, 98511 tokens, paths of up to 8: 47 M 41 us against 52 with a launch a level, 62 M 50 against 60, 77 M 56 against 57;
// what a launch a level takes hardly grows).
constexpr int64_t kAhead = 150LL << 20;
constexpr int64_t kAheadGiven = 75LL << 20;
// Workgroups of the race up to which each of them walks by itself instead of a launch before: 38 (one stream of 152K
// tokens) 17.5 us against 21.4, 988 34.5 against 40.1, 2432 62.7 against 61.8, 4864 68.6 against 60.6.
constexpr int64_t kFused = 3000;
// Nodes of a path that have their own launch: one that no path comes to takes 2 us, a row left to the walk 12.
constexpr int kLevels = 12;

struct Stat {
  float top;   // the slice's largest logit (greedy: the first of them)
  float sum;   // sum of exp2((x - top) log2(e) / temperature); greedy: the index of top, as bits
};

// What the walks leave to the race.
struct State {
  int node;          // the last node of the path (-1: the token is written)
  int count;         // accepted drafts
  uint64_t struck;   // given drafts: the children rejected there, whose tokens are out
  float top, inv_z;  // drawn drafts: the row's softmax,
  float c, c_before; // and the residual, before the last rejection too (where the last is 0 everywhere)
};

struct VerifyArgs {
  const float* logits;
  const float* probs;  // nullable: the drafter's distributions
  const int64_t *draft, *parents;
  const int* plan;
  const float *temperature, *uniforms, *noise;
  int64_t T, V;
  int S, width;  // width: entries of a path
  int slices;
  int64_t *accepted, *path, *tokens;
  State* state;     // [S]
  uint64_t* words;  // [S][slices][2] maxima of the race: after the last rejection, before it
  float* refs;      // [S][slices] what the first of them are relative to: the slices' largest logits
  Stat* stats;      // [T][slices], or of the first levels' nodes [level][S][slices]; null: the walks read the rows
  int* cursors;     // [level][S] the path's nodes (-1: it ends before); null: rows ahead, or none
  int levels;
};

// float -> uint32 with the same order
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
// (larger key, then lower index) is the larger word; 0: nothing
__device__ __forceinline__ uint64_t word_of(float key, uint32_t idx) {
  return static_cast<uint64_t>(order_key(key)) << 32 | ~idx;
}
__device__ __forceinline__ uint32_t index_of(uint64_t word) { return ~static_cast<uint32_t>(word); }
__device__ __forceinline__ float key_of(uint64_t word) {
  const uint32_t u = static_cast<uint32_t>(word >> 32);
  return __builtin_bit_cast(float, (u & 0x80000000u) ? u & 0x7fffffffu : ~u);
}
constexpr uint64_t kBad = ~0ull;  // a row whose softmax is not a number
// A word of the race whose key is relative to a logit `ref`, made relative to one of at least that size.
__device__ __forceinline__ uint64_t shifted(uint64_t word, float ref, float to, float scale) {
  return word == 0 || word == kBad || ref == to ? word : word_of(__builtin_fmaf(ref - to, scale, key_of(word)), index_of(word));
}

__device__ __forceinline__ uint64_t max64(uint64_t a, uint64_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint64_t wave_max64(uint64_t v) {
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) v = max64(v, static_cast<uint64_t>(__shfl_xor(static_cast<long long>(v), d, kWave)));
  return v;
}

__device__ __forceinline__ bool tree_of(const VerifyArgs& a, int s, DraftSeq& u) {
  u = lsh::plan_seqs(a.plan)[s];
  return u.nodes >= 1 && u.nodes <= lsh::kMaxNodes && u.first >= 0 && u.first + u.nodes <= a.T;
}
// This lane's parent in a tree: an earlier node, or -1.
__device__ __forceinline__ int parent_of(const VerifyArgs& a, const DraftSeq& u, int node) {
  const int64_t p = node < u.nodes ? a.parents[u.first + node] : -1;
  return p >= 0 && p < node ? static_cast<int>(p) : -1;
}

// Elements [v0, v0 + 4) of a row, `pad` past its end.
__device__ __forceinline__ f32x4u four(const float* row, int64_t v0, int64_t V, float pad) {
  f32x4u x = {pad, pad, pad, pad};
  if (v0 + 4 <= V) return *reinterpret_cast<const f32x4u*>(row + v0);
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (v0 + e < V) x[e] = row[v0 + e];
  return x;
}

// Elements v0 + 4 STEP i .. + 4 of a row for i = 0 .. N - 1, `pad` past its end. The whole block [base, base +
// 4 STEP N) inside the row is the common case, whose loads have no branch between them.
template <int N, int STEP>
__device__ __forceinline__ void block_of(const float* row, int64_t base, int64_t v0, int64_t V, float pad, f32x4u (&x)[N]) {
  if (base + 4 * STEP * N <= V) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = *reinterpret_cast<const f32x4u*>(row + v0 + i * 4 * STEP);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = four(row, v0 + i * 4 * STEP, V, pad);
  }
}

// argmax with the first index of equal values, NaN above every number
__device__ __forceinline__ uint64_t argmax_word(float x, uint32_t idx) {
  // the positive quiet NaN's key is above infinity's; -0 + 0 is 0
  return word_of(x != x ? __builtin_nanf("") : x + 0.f, idx);
}

// The largest of a thread's elements v0 + 4 STEP i + e below V, as a word; tokens come in growing order.
template <int N, int STEP>
__device__ __forceinline__ uint64_t argmax_part(const f32x4u (&x)[N], int64_t v0, int64_t V) {
  float top = -__builtin_inff();
  uint32_t at = ~0u;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t v = static_cast<uint32_t>(v0 + i * 4 * STEP + e);
      // (a NaN is above every number, and none is above it; the first of a row of -inf counts too)
      const bool up = (x[i][e] > top || (x[i][e] != x[i][e] && top == top) || at == ~0u) && v < V;
      at = up ? v : at;
      top = up ? x[i][e] : top;
    }
  return at == ~0u ? 0 : argmax_word(top, at);
}

// Joins softmax pieces: (top, sum) of two parts, `c` = log2(e) / temperature.
__device__ __forceinline__ void join(float& top, float& sum, float ot, float os, float c) {
  const float m = fmaxf(top, ot);
  if (m == -__builtin_inff()) {  // both parts are empty or all -inf (or NaN, which stays)
    sum += os;
    return;
  }
  sum = (sum == 0.f ? 0.f : sum * __builtin_amdgcn_exp2f((top - m) * c)) + (os == 0.f ? 0.f : os * __builtin_amdgcn_exp2f((ot - m) * c));
  top = m;
}

// A block of N loads of a row: their largest value and the sum of exp2((x - top) c). A NaN gives a NaN sum,
// +infinity too.
template <int N>
__device__ __forceinline__ void softmax_part(const f32x4u (&x)[N], float c, float& top, float& sum) {
  float m = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) m = fmaxf(m, x[i][e]);
  float t = 0.f;
  const float shift = m == -__builtin_inff() ? 0.f : m;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float each = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) each += __builtin_amdgcn_exp2f((x[i][e] - shift) * c);
    t += each;
  }
  top = m;
  sum = t;
}

// ---- rows ahead of the walks --------------------------------------------------------------------

// The workgroup's slice of a row.
__device__ __forceinline__ void slice_of_row(const float* row, int64_t V, int slice, bool greedy, float temp, Stat* out) {
  constexpr int kWaves = kSliceThreads / kWave;
  __shared__ float tops[kWaves], sums[kWaves];
  __shared__ uint64_t words[kWaves];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int64_t base = static_cast<int64_t>(slice) * kSlice, v0 = base + 4 * threadIdx.x;
  f32x4u x[kPer];
  block_of<kPer, kSliceThreads>(row, base, v0, V, -__builtin_inff(), x);
  out += slice;
  if (greedy) {
    const uint64_t best = wave_max64(argmax_part<kPer, kSliceThreads>(x, v0, V));
    if (lane == 0) words[wave] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
      uint64_t all = best;
#pragma unroll
      for (int w = 1; w < kWaves; ++w) all = max64(all, words[w]);
      *reinterpret_cast<uint64_t*>(out) = all;
    }
    return;
  }
  const float c = kLog2e / temp;
  float top, sum;
  softmax_part(x, c, top, sum);
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) join(top, sum, __shfl_xor(top, d, kWave), __shfl_xor(sum, d, kWave), c);
  if (lane == 0) {
    tops[wave] = top;
    sums[wave] = sum;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kWaves; ++w) join(top, sum, tops[w], sums[w], c);
    *out = {top, sum};
  }
}

// A row from its slices, for a whole wavefront.
__device__ __forceinline__ uint64_t argmax_of(const Stat* part, int slices) {
  uint64_t best = 0;
  for (int i = threadIdx.x % kWave; i < slices; i += kWave) best = max64(best, reinterpret_cast<const uint64_t*>(part)[i]);
  return wave_max64(best);
}
__device__ __forceinline__ void softmax_of(const Stat* part, int slices, float c, float& top, float& sum) {
  top = -__builtin_inff();
  sum = 0.f;
  for (int i = threadIdx.x % kWave; i < slices; i += kWave) join(top, sum, part[i].top, part[i].sum, c);
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) join(top, sum, __shfl_xor(top, d, kWave), __shfl_xor(sum, d, kWave), c);
}

__global__ __launch_bounds__(kSliceThreads) void row_stats_kernel(VerifyArgs a) {
  const int64_t t = blockIdx.x;
  const int s = a.plan[lsh::plan_owners_at(a.S) + t];
  if (s < 0 || s >= a.S) return;
  DraftSeq u;
  if (!tree_of(a, s, u)) return;
  const float temp = a.temperature[s];
  const bool greedy = temp < 1e-5f;
  const int node = static_cast<int>(t) - u.first;
  if (!greedy && __ballot(parent_of(a, u, threadIdx.x % kWave) == node) == 0) return;  // nothing is tested there
  slice_of_row(a.logits + t * a.V, a.V, blockIdx.y, greedy, temp, a.stats + t * a.slices);
}

// What the tokens of the lanes in `struck` leave of a row's softmax, for a whole wavefront: a sum over all others.
__device__ __forceinline__ double mass_of(const float* row, int64_t V, int64_t tok, uint64_t struck, float c, float top, float inv_z) {
  constexpr int N = 4;
  double sum = 0.0;
  for (int64_t base = 0; base < V; base += 4 * N * kWave) {
    const int64_t v0 = base + 4 * (threadIdx.x % kWave);
    f32x4u x[N];
    block_of<N, kWave>(row, base, v0, V, -__builtin_inff(), x);
    for (uint64_t todo = __ballot(tok >= base && tok < base + 4 * N * kWave) & struck; todo; todo &= todo - 1) {
      const int64_t at = __shfl(static_cast<long long>(tok), __builtin_ctzll(todo), kWave) - v0;
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[i][e] = at == 4 * kWave * i + e ? -__builtin_inff() : x[i][e];
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) sum += static_cast<double>(__builtin_amdgcn_exp2f((x[i][e] - top) * c)) * inv_z;
  }
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) sum += __shfl_xor(sum, d, kWave);
  return sum;
}

// A lane's node as the tests of given drafts see it: `child` of the node, its token (-1: none), number and
// probability (exp2((logit - top) c) inv_z of the node's row). The first of `children` that is accepted, or -1;
// `struck`: the rejected ones, whose tokens are out.
// What is left of p is 1 less the struck tokens' p, while that is far from their roundings (under 2^-20 together);
// below kSure it is summed: a walk gets there with a probability of no more than kSure. So a token that has all that is
// left has r = 1 and is taken, and one that is not 0 remains for the race.
constexpr double kSure = 0x1p-14;
__device__ __forceinline__ int take_given(uint64_t children, bool child, int64_t tok, float unif, double p_own, const float* row,
                                          int64_t V, float c, float top, float inv_z, uint64_t& struck) {
  double left = 1.0;  // what the struck tokens left of p
  struck = 0;
  for (uint64_t todo = children; todo; todo &= todo - 1) {
    const int i = __builtin_ctzll(todo);
    const double p = __shfl(p_own, i, kWave), number = static_cast<double>(__shfl(unif, i, kWave));
    const int64_t t = __shfl(static_cast<long long>(tok), i, kWave);
    const bool again = (__ballot(child && tok == t) & struck) != 0;  // struck already
    if (number < (again ? 0.0 : p / left)) return i;
    if (t < 0 || !(p > 0.0) || again) continue;
    double rest = left - p;
    if (rest < kSure) rest = mass_of(row, V, tok, struck | 1ull << i, c, top, inv_z);
    if (!(rest > 0.0)) {  // the token has all of it
      if (number < 1.0) return i;
      continue;
    }
    left = rest;
    struck |= 1ull << i;
  }
  return -1;
}

// Node `level` of the paths of given drafts: the step there from the node before, and a slice of its row.
__global__ __launch_bounds__(kSliceThreads) void level_kernel(VerifyArgs a, int level) {
  const int s = blockIdx.y, lane = threadIdx.x % kWave;
  DraftSeq u;
  if (!tree_of(a, s, u)) return;
  const float temp = a.temperature[s];
  const bool greedy = temp < 1e-5f;
  const int par = parent_of(a, u, lane);
  int node = 0;
  if (level > 0) {
    const int before = a.cursors[(level - 1) * a.S + s];
    node = -1;
    if (before >= 0) {
      const Stat* part = a.stats + ((level - 1) * static_cast<int64_t>(a.S) + s) * a.slices;
      const bool child = par == before;
      const uint64_t children = level < a.width ? __ballot(child) : 0;
      int64_t tok = child ? a.draft[u.first + lane] : -1;
      if (tok >= a.V) tok = -1;
      if (greedy) {
        const int64_t best = index_of(argmax_of(part, a.slices));
        const uint64_t hit = __ballot(child && tok == best) & children;
        if (hit) node = __builtin_ctzll(hit);
      } else if (children) {
        const float c = kLog2e / temp, unif = child ? a.uniforms[u.first + lane] : 0.f;
        const float xl = tok >= 0 ? a.logits[(u.first + before) * a.V + tok] : -__builtin_inff();
        float top, sum;
        softmax_of(part, a.slices, c, top, sum);
        const float inv_z = 1.f / sum;
        uint64_t struck;
        node = take_given(children, child, tok, unif,
                          tok >= 0 ? static_cast<double>(__builtin_amdgcn_exp2f((xl - top) * c)) * inv_z : 0.0,
                          a.logits + (u.first + before) * a.V, a.V, c, top, inv_z, struck);
      }
    }
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) a.cursors[level * a.S + s] = node;
  if (node < 0) return;
  if (!greedy && (level + 1 >= a.width || __ballot(par == node) == 0)) return;  // nothing is tested there
  slice_of_row(a.logits + (u.first + node) * a.V, a.V, blockIdx.x, greedy, temp,
               a.stats + (level * static_cast<int64_t>(a.S) + s) * a.slices);
}

// ---- the walks ------------------------------------------------------------------------------------

// What the first wavefront of a walk asks its workgroup for, and each wavefront's part of the answer.
enum Pass { kDone, kArgmax, kSoftmax, kResidual };
template <int WAVES>
struct Shared {
  int pass, node;
  float top, inv_z, c;  // kResidual
  uint64_t words[WAVES];
  float tops[WAVES], sums[WAVES];
  double parts[WAVES];
};

// This wavefront's part of a pass over a row by a workgroup of WAVES.
template <int WAVES>
__device__ __forceinline__ void part_of_pass(const VerifyArgs& a, const DraftSeq& u, Shared<WAVES>& sh, int pass, int node,
                                             float scale) {
  constexpr int THREADS = WAVES * kWave;
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const float* row = a.logits + (u.first + node) * a.V;
  if (pass == kArgmax) {
    constexpr int N = 8;  // 16-byte loads in flight for each thread
    uint64_t best = 0;
    for (int64_t base = 0; base < a.V; base += 4 * N * THREADS) {
      const int64_t v0 = base + 4 * tid;
      f32x4u x[N];
      block_of<N, THREADS>(row, base, v0, a.V, -__builtin_inff(), x);
      best = max64(best, argmax_part<N, THREADS>(x, v0, a.V));
    }
    best = wave_max64(best);
    if (lane == 0) sh.words[wave] = best;
  } else if (pass == kSoftmax) {
    constexpr int N = 8;
    float top = -__builtin_inff(), sum = 0.f;
    for (int64_t base = 0; base < a.V; base += 4 * N * THREADS) {
      f32x4u x[N];
      block_of<N, THREADS>(row, base, base + 4 * tid, a.V, -__builtin_inff(), x);
      float t, z;
      softmax_part(x, scale, t, z);
      join(top, sum, t, z, scale);
    }
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) join(top, sum, __shfl_xor(top, d, kWave), __shfl_xor(sum, d, kWave), scale);
    if (lane == 0) {
      sh.tops[wave] = top;
      sh.sums[wave] = sum;
    }
  } else {
    constexpr int N = 4;
    const float* qr = a.probs + (u.first + node) * a.V;
    const float top = sh.top, inv_z = sh.inv_z, c = sh.c;
    double part = 0.0;
    for (int64_t base = 0; base < a.V; base += 4 * N * THREADS) {
      f32x4u x[N], y[N];
      block_of<N, THREADS>(row, base, base + 4 * tid, a.V, -__builtin_inff(), x);
      block_of<N, THREADS>(qr, base, base + 4 * tid, a.V, 0.f, y);
      float some = 0.f;
#pragma unroll
      for (int j = 0; j < N; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          some += fmaxf(__builtin_fmaf(-c, y[j][e], __builtin_amdgcn_exp2f((x[j][e] - top) * scale) * inv_z), 0.f);
      part += static_cast<double>(some);
    }
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) part += __shfl_xor(part, d, kWave);
    if (lane == 0) sh.parts[wave] = part;
  }
}

// A wavefront walks a sequence's tree. PASSES: the other wavefronts of its workgroup (of WAVES) wait in
// help() for the rows it has to read (without: there are none). `write`: the result goes to memory.
template <int WAVES, bool PASSES>
__device__ __forceinline__ State walk(const VerifyArgs& a, int s, Shared<WAVES>& sh, bool write) {
  const int lane = threadIdx.x % kWave;
  DraftSeq u;
  const bool valid = tree_of(a, s, u);
  int64_t* path = a.path + static_cast<int64_t>(s) * a.width;
  int64_t* tokens = a.tokens + static_cast<int64_t>(s) * a.width;
  State st{};
  st.node = -1;
  if (!valid) {
    if (write) {
      for (int j = lane; j < a.width; j += kWave) path[j] = tokens[j] = -1;
      if (lane == 0) a.accepted[s] = 0;
    }
    return st;
  }
  const float temp = a.temperature[s];
  const bool greedy = temp < 1e-5f;
  const float c = kLog2e / temp;
  auto ask = [&](int pass, int node) {
    if constexpr (PASSES) {
      if (lane == 0) {
        sh.pass = pass;
        sh.node = node;
      }
      if (WAVES > 1) __syncthreads();  // everyone starts
      part_of_pass<WAVES>(a, u, sh, pass, node, c);
      if (WAVES > 1) __syncthreads();  // everyone is done
    }
  };
  // ---- this lane's node: its parent, token, number, and the parent's logit and q of the token
  const int par = parent_of(a, u, lane);
  int64_t tok = -1;
  float unif = 0.f, xl = -__builtin_inff(), ql = 0.f;
  if (par >= 0) {
    tok = a.draft[u.first + lane];
    unif = a.uniforms[u.first + lane];
    if (tok >= a.V) tok = -1;
    if (tok >= 0 && !greedy) {
      const int64_t at = (u.first + par) * a.V + tok;
      xl = a.logits[at];
      if (a.probs) ql = a.probs[at];
    }
  }
  int node = 0, count = 0;
  uint64_t on_path = 1;
  int64_t last = -1;
  if (a.cursors) {  // nodes of the path that levels took
    const int at = lane < a.levels ? a.cursors[lane * a.S + s] : -1;
    const uint64_t there = __ballot(at >= 0);  // (node 0 is)
    const int known = __builtin_popcountll(there);
    count = known - 1;
    for (int l = 1; l < known; ++l) {
      node = __shfl(at, l, kWave);
      on_path |= 1ull << node;
    }
  }
  while (true) {  // each round but the last adds a node to the path
    // this node's slices, where there are any
    const Stat* const part = !a.stats      ? nullptr
                             : !a.cursors  ? a.stats + (u.first + node) * static_cast<int64_t>(a.slices)
                             : count < a.levels ? a.stats + (count * static_cast<int64_t>(a.S) + s) * a.slices
                                                : nullptr;
    const uint64_t all = __ballot(par == node);
    uint64_t children = count + 1 < a.width ? all : 0;
    int taken = -1;
    if (greedy) {
      uint64_t best = 0;
      if (!PASSES || part) {
        best = argmax_of(part, a.slices);
      } else {
        ask(kArgmax, node);
        for (int w = 0; w < WAVES; ++w) best = max64(best, sh.words[w]);
      }
      last = index_of(best);
      const uint64_t hit = __ballot(par == node && tok == last) & children;
      if (hit) taken = __builtin_ctzll(hit);
    } else if (children) {
      float top = -__builtin_inff(), sum = 0.f;
      if (!PASSES || part) {
        softmax_of(part, a.slices, c, top, sum);
      } else {
        ask(kSoftmax, node);
        for (int w = 0; w < WAVES; ++w) join(top, sum, sh.tops[w], sh.sums[w], c);
      }
      const float inv_z = 1.f / sum;
      const double p_own = par == node && tok >= 0 ? static_cast<double>(__builtin_amdgcn_exp2f((xl - top) * c)) * inv_z : 0.0;
      st.top = top;
      st.inv_z = inv_z;
      st.struck = 0;
      st.c = st.c_before = 0.f;
      if (a.probs == nullptr)
        taken = take_given(children, par == node, tok, unif, p_own, a.logits + (u.first + node) * a.V, a.V, c, top, inv_z, st.struck);
      double rc = 0.0, rn = 1.0;  // drawn drafts: r = (p - rc q)+ / rn
      for (uint64_t todo = PASSES && a.probs ? children : 0; todo && taken < 0; todo &= todo - 1) {
        const int i = __builtin_ctzll(todo);
        const double p = __shfl(p_own, i, kWave), number = static_cast<double>(__shfl(unif, i, kWave));
        const int64_t t = __shfl(static_cast<long long>(tok), i, kWave);
        const double q = static_cast<double>(__shfl(ql, i, kWave));
        const double d = p - rc * q, r = (d > 0.0 || d != d ? d : 0.0) / rn;
        if (t >= 0 && number * q < r) {
          taken = i;
          continue;
        }
        const double next = rc + rn;
        if (todo & (todo - 1)) {  // another child is tested against what is left
          if (lane == 0) {
            sh.top = top;
            sh.inv_z = inv_z;
            sh.c = static_cast<float>(next);
          }
          ask(kResidual, node);
          double left = sh.parts[0];
          for (int w = 1; w < WAVES; ++w) left += sh.parts[w];
          if (left > 0.0) {
            rc = next;
            rn = left;
            st.c_before = st.c;
            st.c = static_cast<float>(rc);
          }
        } else {
          st.c_before = st.c;
          st.c = static_cast<float>(next);
        }
      }
    }
    if (a.cursors && count + 1 < a.levels) taken = -1;  // (what the level after this one found, as it found it)
    if (taken < 0) {
      if (!children) {  // nothing was rejected here
        st.struck = 0;
        st.c = st.c_before = 0.f;
      }
      break;
    }
    node = taken;
    on_path |= 1ull << taken;
    ++count;
  }
  st.node = greedy ? -1 : node;
  st.count = count;
  if (!write) return st;
  // ---- the path: a lane writes its own node's place
  for (int j = lane; j < a.width; j += kWave) {
    if (j > count) path[j] = -1;
    if (j > count || (j == count && !greedy)) tokens[j] = -1;
  }
  if (on_path >> lane & 1) {
    const int at = __builtin_popcountll(on_path & ((1ull << lane) - 1));  // (a path's nodes grow)
    path[at] = lane;
    if (at > 0) tokens[at - 1] = a.draft[u.first + lane];
  }
  if (lane == 0) {
    a.accepted[s] = count;
    if (greedy) tokens[count] = last < a.V ? last : 0;
  }
  return st;
}

// The other wavefronts of a walk's workgroup.
template <int WAVES>
__device__ __forceinline__ void help(const VerifyArgs& a, int s, Shared<WAVES>& sh) {
  DraftSeq u;
  tree_of(a, s, u);
  const float scale = kLog2e / a.temperature[s];
  while (true) {
    __syncthreads();
    const int pass = sh.pass;
    if (pass == kDone) return;
    part_of_pass<WAVES>(a, u, sh, pass, sh.node, scale);
    __syncthreads();
  }
}

// A workgroup for a sequence. One wavefront decides, the others read rows with it (all 16 deciding the same, on one CU,
// took 46 us for 32 chains with probabilities and 63 for 24 large trees, the whole call; this 42 and 59).
template <int WAVES>
__global__ __launch_bounds__(WAVES* kWave) void walk_kernel(VerifyArgs a) {
  __shared__ Shared<WAVES> sh;
  const int s = blockIdx.x;
  if (WAVES > 1 && __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave) != 0) {
    help<WAVES>(a, s, sh);
    return;
  }
  const State st = walk<WAVES, true>(a, s, sh, true);
  if (threadIdx.x == 0) {
    a.state[s] = st;
    sh.pass = kDone;
  }
  if (WAVES > 1) __syncthreads();
}

// ---- the race for the last token -------------------------------------------------------------------

// WALK: every workgroup of a slice walks the tree by itself, while its part of the noise is under way.
template <bool WALK>
__global__ __launch_bounds__(kSliceThreads) void race_kernel(VerifyArgs a) {
  constexpr int kWaves = kSliceThreads / kWave;
  __shared__ uint64_t words[2][kWaves];
  __shared__ float tops[kWaves];
  __shared__ Shared<1> none;
  __shared__ State walked;
  __shared__ uint32_t out[kSlice / 32];  // bits: struck tokens of the slice
  const int s = blockIdx.y, tid = threadIdx.x, lane = tid % kWave;
  const float* noise = a.noise + static_cast<int64_t>(s) * a.V;
  const int64_t base = static_cast<int64_t>(blockIdx.x) * kSlice, v0 = base + 4 * tid;
  f32x4u e[kPer];
  if constexpr (WALK) {
    block_of<kPer, kSliceThreads>(noise, base, v0, a.V, 1.f, e);
    if (__builtin_amdgcn_readfirstlane(tid / kWave) == 0) {
      const State st = walk<1, false>(a, s, none, blockIdx.x == 0);
      if (lane == 0) {
        walked = st;
        if (blockIdx.x == 0) a.state[s] = st;
      }
    }
    __syncthreads();
  }
  const State* const state = WALK ? &walked : a.state + s;
  const int node = state->node;
  if (node < 0) return;
  const DraftSeq u = lsh::plan_seqs(a.plan)[s];
  const uint64_t struck = state->struck;
  const float c = state->c, c_before = state->c_before, top = state->top, inv_z = state->inv_z;
  const float scale = kLog2e / a.temperature[s];
  const float* row = a.logits + (u.first + node) * a.V;
  const bool drawn = !WALK && a.probs != nullptr && c > 0.f;
  f32x4u x[kPer], q[kPer];
  block_of<kPer, kSliceThreads>(row, base, v0, a.V, -__builtin_inff(), x);
  if constexpr (!WALK) block_of<kPer, kSliceThreads>(noise, base, v0, a.V, 1.f, e);
  if (drawn) block_of<kPer, kSliceThreads>(a.probs + (u.first + node) * a.V, base, v0, a.V, 0.f, q);
  if (struck) {
    for (int i = tid; i < kSlice / 32; i += kSliceThreads) out[i] = 0;
    __syncthreads();
    if (tid < kWave && (struck >> lane & 1)) {
      const int64_t t = a.draft[u.first + lane] - base;
      if (t >= 0 && t < kSlice) atomicOr(&out[t / 32], 1u << (t % 32));
    }
    __syncthreads();
  }
  // the largest logit of the wavefront's part (one that is not finite: 0, and the row is bad or the part empty)
  float ref = 0.f;
  if (!drawn) {
    ref = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < kPer; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) ref = fmaxf(ref, x[i][j]);
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) ref = fmaxf(ref, __shfl_xor(ref, d, kWave));
    ref = fabsf(ref) < __builtin_inff() ? ref : 0.f;
  }
  // this thread's largest key and its token, the first of equal ones (tokens come in growing order)
  float key = -__builtin_inff(), key_before = -__builtin_inff();
  uint32_t at = 0, at_before = 0;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int64_t v = v0 + i * 4 * kSliceThreads;
    uint32_t gone = 0;
    if (struck) gone = out[(v - base) / 32] >> ((v - base) % 32);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t idx = static_cast<uint32_t>(v + j);
      const float lg_e = __builtin_amdgcn_logf(fmaxf(e[i][j], 1.17549435e-38f));  // log2
      bad |= !(x[i][j] < __builtin_inff());  // NaN or infinite: the softmax is no number
      if (drawn) {
        const float p = __builtin_amdgcn_exp2f((x[i][j] - top) * scale) * inv_z;
        const float r = __builtin_fmaf(-c, q[i][j], p), r0 = __builtin_fmaf(-c_before, q[i][j], p);
        const float k = r > 0.f ? __builtin_amdgcn_logf(r) - lg_e : -__builtin_inff();
        const float k0 = r0 > 0.f ? __builtin_amdgcn_logf(r0) - lg_e : -__builtin_inff();
        at = k > key ? idx : at;
        key = fmaxf(key, k);
        at_before = k0 > key_before ? idx : at_before;
        key_before = fmaxf(key_before, k0);
      } else {
        const float k = gone >> j & 1 ? -__builtin_inff() : __builtin_fmaf(x[i][j] - ref, scale, -lg_e);
        at = k > key ? idx : at;
        key = fmaxf(key, k);
      }
    }
  }
  uint64_t best = key > -__builtin_inff() ? word_of(key, at) : 0;
  uint64_t before = key_before > -__builtin_inff() ? word_of(key_before, at_before) : 0;
  if (bad) best = kBad;
  best = wave_max64(best);
  before = wave_max64(before);
  if (lane == 0) {
    words[0][tid / kWave] = best;
    words[1][tid / kWave] = before;
    tops[tid / kWave] = best ? ref : -__builtin_inff();
  }
  __syncthreads();
  if (tid != 0) return;
  float top_ref = tops[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) top_ref = fmaxf(top_ref, tops[w]);
  best = shifted(best, tops[0], top_ref, scale);
#pragma unroll
  for (int w = 1; w < kWaves; ++w) {
    best = max64(best, shifted(words[0][w], tops[w], top_ref, scale));
    before = max64(before, words[1][w]);
  }
  const int64_t at_slice = static_cast<int64_t>(s) * a.slices + blockIdx.x;
  a.words[2 * at_slice] = best;
  a.words[2 * at_slice + 1] = before;
  a.refs[at_slice] = top_ref;
}

// Joins the slices: a wavefront for each sequence.
__global__ __launch_bounds__(kWave) void finish_kernel(VerifyArgs a) {
  const int s = blockIdx.x, lane = threadIdx.x;
  const State* const state = a.state + s;
  if (state->node < 0) return;
  const uint64_t* words = a.words + static_cast<int64_t>(s) * a.slices * 2;
  const float* refs = a.refs + static_cast<int64_t>(s) * a.slices;
  const float scale = kLog2e / a.temperature[s];
  uint64_t best = 0, before = 0;  // of this lane's slices
  float ref = -__builtin_inff();  // what best is relative to
  for (int i = lane; i < a.slices; i += kWave) {
    const float other = refs[i], to = fmaxf(ref, other);
    best = max64(shifted(best, ref, to, scale), shifted(words[2 * i], other, to, scale));
    ref = to;
    before = max64(before, words[2 * i + 1]);
  }
  float top = ref;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) top = fmaxf(top, __shfl_xor(top, d, kWave));
  best = shifted(best, ref, top, scale);
  best = wave_max64(best);
  before = wave_max64(before);
  const uint64_t word = best ? best : before;
  const uint32_t idx = index_of(word);
  if (lane == 0)
    a.tokens[static_cast<int64_t>(s) * a.width + state->count] = word == 0 || word == kBad || idx >= a.V ? 0 : idx;
}

int64_t slices_of(int64_t V) { return (V + kSlice - 1) / kSlice; }

}  // namespace

extern "C" int64_t llmserve_verify_draft_workspace_bytes(int64_t S, int64_t T, int64_t V) {
  if (S <= 0 || T < 0 || V <= 0) return 0;
  return S * static_cast<int64_t>(sizeof(State)) + S * slices_of(V) * (16 + static_cast<int64_t>(sizeof(float))) + 8 +
         std::max(T * V <= kAhead ? T * slices_of(V) * static_cast<int64_t>(sizeof(Stat)) : 0,
                  T * V > kAheadGiven ? kLevels * S * (slices_of(V) * static_cast<int64_t>(sizeof(Stat)) + 4) : 0);
}

extern "C" int llmserve_verify_draft(const float* logits, const int64_t* draft_tokens, const int64_t* parents,
                                     const void* plan, const float* temperature, const float* uniforms,
                                     const float* noise, const float* draft_probs, int64_t S, int64_t T, int64_t V,
                                     int64_t max_depth, int64_t* accepted, int64_t* path, int64_t* tokens,
                                     void* workspace, int64_t workspace_bytes, void* stream) {
  LSH_CHECK(S >= 0 && T >= 0 && V >= 1 && V < (1LL << 24), "verify_draft: 1 <= V < 2^24 (got %lld)", (long long)V);
  LSH_CHECK(max_depth >= 0 && max_depth < lsh::kMaxNodes, "verify_draft: max_depth %lld not in [0, 63]",
            (long long)max_depth);
  if (S == 0) return LLMSERVE_OK;
  LSH_CHECK(S < (1 << 16) && T < (1LL << 24), "verify_draft: batch too large");
  LSH_CHECK(plan && temperature && noise && accepted && path && tokens &&
                (T == 0 || (logits && draft_tokens && parents && uniforms)),
            "verify_draft: null pointer");
  const int64_t need = llmserve_verify_draft_workspace_bytes(S, T, V);
  LSH_CHECK(workspace != nullptr && workspace_bytes >= need && lsh::aligned16(workspace),
            "verify_draft: a 16-byte aligned workspace of %lld bytes is needed (%lld given)", (long long)need,
            (long long)workspace_bytes);
  const int64_t slices = slices_of(V);
  State* const state = static_cast<State*>(workspace);
  uint64_t* const words = reinterpret_cast<uint64_t*>(state + S);
  const bool ahead = T * V <= (draft_probs ? kAhead : kAheadGiven), by_level = !ahead && draft_probs == nullptr;
  const int levels = static_cast<int>(max_depth + 1 < kLevels ? max_depth + 1 : kLevels);
  float* const refs = reinterpret_cast<float*>(words + S * slices * 2);
  Stat* const stats = reinterpret_cast<Stat*>(refs + (S * slices + 1) / 2 * 2);  // (8-byte words in greedy rows)
  const VerifyArgs a{logits, draft_probs, draft_tokens, parents, static_cast<const int*>(plan), temperature, uniforms, noise,
               T, V, static_cast<int>(S), static_cast<int>(max_depth + 1), static_cast<int>(slices),
               accepted, path, tokens, state,
               words, refs, ahead || by_level ? stats : nullptr,
               by_level ? reinterpret_cast<int*>(stats + levels * S * slices) : nullptr, levels};
  hipStream_t st = lsh::as_stream(stream);
  const unsigned n = static_cast<unsigned>(S), parts = static_cast<unsigned>(slices);
  if (ahead && T > 0)
    lsh::launch(row_stats_kernel, dim3(static_cast<unsigned>(T), parts), dim3(kSliceThreads), 0, st, false, a);
  for (int level = 0; by_level && level < levels; ++level)
    lsh::launch(level_kernel, dim3(parts, n), dim3(kSliceThreads), 0, st, false, a, level);
  const bool slices_only = draft_probs == nullptr && (ahead || levels > max_depth);  // the walks read no row
  if (slices_only && S * slices <= kFused) {
    lsh::launch(race_kernel<true>, dim3(parts, n), dim3(kSliceThreads), 0, st, false, a);
  } else {
    // (a wavefront is enough where no row is left to read)
    if (slices_only)
      lsh::launch(walk_kernel<1>, dim3(n), dim3(kWave), 0, st, false, a);
    else
      lsh::launch(walk_kernel<kWalkWaves>, dim3(n), dim3(kWalkWaves * kWave), 0, st, false, a);
    lsh::launch(race_kernel<false>, dim3(parts, n), dim3(kSliceThreads), 0, st, false, a);
  }
  lsh::launch(finish_kernel, dim3(n), dim3(kWave), 0, st, true, a);
  return lsh::launch_status("verify_draft");
}
