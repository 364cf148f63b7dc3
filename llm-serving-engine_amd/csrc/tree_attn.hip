// Attention of drafted tokens over the paged cache: node i of a sequence's tree sees the cached
// tokens and, of the tree's own ones, its ancestors and itself (draft.h, draft_meta.hip):
//   s_t = scale (q' . k_t),  out = sum_t softmax(s)_t v_t  over t < ctx and t = ctx + j, j in ancestors(i)
//   q' = q_mult ? q * q_mult : q;  k_t, v_t the cache rows (int8 codes times their fp32 scales, or fp32)
// Tokens whose block id lies outside the cache add nothing; a node that sees no token gives NaN.
//
// All nodes of a tree and all query heads of a kv head read the same tokens, so the (node, head) pairs
// are the rows of two matrix products and the cache is read once for all of them. A workgroup takes
// one kv head and a block of the plan's line (draft.h): parts of one or more tiles of up to 128 rows. Its four
// wavefronts are split over the rows, 32 for each, and where there are at most 64 or 32 rows over the
// tokens, two or four ways. Parts of a tile that several workgroups have are joined by a second launch.
//
// Both products are transposed: S^T = K Q^T leaves lane (fr, fc) the scores of row fr for tokens
// 4 fc + e of every 16, which is the B operand of O^T = V^T P^T when that product's k order is those
// tokens. K needs no transposition (a lane reads a quarter of its token's row, the dims of a product step
// being any four groups of the row's), V's is done by byte permutes in registers (int8) or is none
// at all (fp32: one register is one element). A row's running reference and sum are per-lane scalars.
//
// Precision is fp32's. int8: the scores are exact integer products of the codes with q in three signed digits (23 bits of
// the row's largest element), or where few elements come near that one, of codes in fp16 with q in two fp16 pieces. Codes
// of V are exact in fp16, the weights two fp16 pieces after scaling by a power of two (22 bits); scales stay in fp32 on
// the score and the weight. fp32: fp32
// matrix instructions (a step's sums formed apart and added once), for a head size of 128 and more than 32 rows a
// tree on average fp16 ones on two pieces of everything: 22 bits of every element down to 2^-29 of its row's largest.
// Errors against 64 bits lie between 2e-7 and 4.5e-7 of the 2-norm, and with channels of very different size below 2e-6 of
// each channel's.
//
// What bounds it. int8, 32 trees of up to 64 nodes over 1K to 8K tokens (1716 nodes, 16 heads, 8 of K/V, D 128, 55 GFLOP,
// 298 MB): 168 us, 330 TFLOP/s; vector instructions (13 for each score of a lane, 80 to widen V) are issued in 64 % of the
// SIMDs' cycles, the matrix unit is busy in 31 %, hidden behind them. 16 trees of 26 nodes: 46 us, 1.9 TB/s: 22 us
// of tiles, the rest the starts and ends of the workgroups (plan, table, q: 8 us, joining 4 us) and the second launch
// (61 % and 21 %). One stream: 16 us of kernels, two launches and one tile. Single tokens of 64
// sequences over 2K tokens: 78 us, 3.5 TB/s. fp32: 32 sequences of 5 nodes (10 rows) over 1K to 4K tokens 136 us, 4.9 TB/s; 208
// rows a kv head 46 us (95 TFLOP/s) in fp16 pieces, vector instructions in 49 %, products in 18 % of the cycles. D 64, 16
// trees of 26 nodes over 512 to 4K tokens, 8 kv heads: int8 29 us, 1.5 TB/s, fp32 46 us, 3.5 TB/s.
#include <algorithm>
#include <type_traits>

#include "draft.h"

namespace {

using lsh::DraftItem;
using lsh::DraftSeq;
using lsh::kWave;
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWaves = 4;
constexpr int kCols = 2;                   // 16-row tiles of a wavefront
constexpr int kWaveRows = 16 * kCols;
constexpr int64_t kSplitRows = 32;
static_assert(kWaves * kWaveRows == lsh::kTreeRows);
// Weights: p = exp2(score - ref), the reference moving only when a score passes it by kLazy. int8: ref is
// the running max of score + log2(v scale) - kTop, so that p v_scale lies near the top of fp16's range and
// below 2^(kTop + kLazy). A v scale below 2^(kTop - kMaxLv) counts as that: p stays below 2^(kMaxLv + kLazy),
// whose sum over 2^21 tokens fp32 holds.
constexpr float kLazy = 4.f, kTop = 4.f, kMaxLv = 100.f;

struct TreeArgs {
  const float* q;
  const void* kc;
  const void* vc;
  const float* ks;
  const float* vs;
  const int64_t* bt;
  const int64_t* ancestors;
  const int* plan;
  const float* q_mult;
  float* out;
  float* part_acc;  // [item][kv head][row of the tile][D]
  float* part_rl;   // [item][kv head][row of the tile][2] (reference, sum)
  int64_t num_slots;
  int64_t T;
  int S, Hq, Hk, G, max_blocks, bs, bs_shift;  // bs_shift: log2(bs), or -1
  int items;                                   // capacity of the plan
  float scale;
};

__device__ __forceinline__ f16x2 as_h2(uint32_t w) { return __builtin_bit_cast(f16x2, w); }
__device__ __forceinline__ uint32_t as_u(f16x2 h) { return __builtin_bit_cast(uint32_t, h); }

// Max over the lanes with the same lane % 16.
__device__ __forceinline__ float max_over_fc(float v) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  v = fmaxf(__builtin_bit_cast(float, static_cast<uint32_t>(a[0])), __builtin_bit_cast(float, static_cast<uint32_t>(a[1])));
  const uint32_t w = __builtin_bit_cast(uint32_t, v);
  const auto b = __builtin_amdgcn_permlane16_swap(w, w, false, false);
  return fmaxf(__builtin_bit_cast(float, static_cast<uint32_t>(b[0])), __builtin_bit_cast(float, static_cast<uint32_t>(b[1])));
}
__device__ __forceinline__ float sum_over_fc(float v) {
  v += __shfl_xor(v, 16, kWave);
  return v + __shfl_xor(v, 32, kWave);
}

// `v` of another lane of the same 16, by a data-parallel-primitive control.
template <int CTRL>
__device__ __forceinline__ float row_lane(float v) {
  const int u = __builtin_bit_cast(int, v);
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(u, u, CTRL, 0xf, 0xf, false));
}

// a x and b y -> packed hi and lo pieces (the empty asm makes hi one value: see prefill_attn.hip).
__device__ __forceinline__ void split2(float a, float x, float b, float y, uint32_t& hi, uint32_t& lo) {
  hi = as_u(f16x2{static_cast<_Float16>(__builtin_fmaf(a, x, -0.f)), static_cast<_Float16>(__builtin_fmaf(b, y, -0.f))});
  asm("" : "+v"(hi));
  const f16x2 h = as_h2(hi);
  lo = as_u(f16x2{static_cast<_Float16>(__builtin_fmaf(a, x, -static_cast<float>(h[0]))),
                  static_cast<_Float16>(__builtin_fmaf(b, y, -static_cast<float>(h[1])))});
}

// The same with the low pieces 2^11 times as large (a low piece is up to 2^-12 of its high one): rounded to their smallest
// step, 2^-24, they are off by 2^-36, which is 2^-22 of the smallest high piece that is a normal number.
constexpr float kLoUp = 2048.f;
__device__ __forceinline__ void split2_up(float a, float x, float b, float y, uint32_t& hi, uint32_t& lo) {
  hi = as_u(f16x2{static_cast<_Float16>(__builtin_fmaf(a, x, -0.f)), static_cast<_Float16>(__builtin_fmaf(b, y, -0.f))});
  asm("" : "+v"(hi));
  const f16x2 h = as_h2(hi);
  const float r0 = __builtin_fmaf(a, x, -static_cast<float>(h[0])), r1 = __builtin_fmaf(b, y, -static_cast<float>(h[1]));
  lo = as_u(f16x2{static_cast<_Float16>(r0 * kLoUp), static_cast<_Float16>(r1 * kLoUp)});
}

// Byte J of two words, each a value + 128 -> the two values times 2^-9 in fp16, exact. A byte alone is that many
// of fp16's smallest steps of 2^-24. (The matrix instructions would take those as they are, but align the
// products by their exponents as written: 2e-6 of the result were lost.)
template <int J>
__device__ __forceinline__ uint32_t bytes_to_h2(uint32_t x0, uint32_t x1) {
  const f16x2 up = {32768, 32768}, zero = {-0.25, -0.25};
  return as_u(__builtin_elementwise_fma(as_h2(__builtin_amdgcn_perm(x1, x0, 0x0c040c00u + 0x10001u * J)), up, zero));
}
constexpr float kVUp = 512.f;
// Four int8 codes of a word, in order, as two words of fp16, times 2^-9.
__device__ __forceinline__ u32x2 codes_to_h2(uint32_t codes) {
  const f16x2 up = {32768, 32768}, zero = {-0.25, -0.25};
  const uint32_t x = codes ^ 0x80808080u;
  return u32x2{as_u(__builtin_elementwise_fma(as_h2(__builtin_amdgcn_perm(x, x, 0x0c010c00u)), up, zero)),
               as_u(__builtin_elementwise_fma(as_h2(__builtin_amdgcn_perm(x, x, 0x0c030c02u)), up, zero))};
}

// What a wavefront of a workgroup computes.
struct Work {
  int seq, first, ctx, ranges;  // the sequence, its first node's row of the stream, its cached tokens, its ranges
  int row0, rows;               // rows [row0, row0 + rows) of the tree's nodes * G
  int RW, rw, TW, tw;           // row groups, this wavefront's; shares of the steps, this wavefront's
  int rw_bits, tw_bits;         // log2 of RW, TW
  int t0, t1;                   // positions
  int kvh;
};

// False: nothing to compute (the same for the whole workgroup).
__device__ __forceinline__ bool work_of(const TreeArgs& a, int kvh, int item, int wave, Work& w) {
  const auto* p = reinterpret_cast<const i32x4*>(lsh::plan_items(a.plan, a.S, a.T) + min(item, a.items - 1));
  const i32x4 lo = p[0], hi = p[1];
  auto uniform = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
  w.seq = uniform(lo[0]);
  const int tile = uniform(lo[1]), nodes = min(uniform(hi[1]), lsh::kMaxNodes);
  w.first = uniform(hi[0]);
  w.ctx = uniform(hi[2]);
  w.ranges = uniform(hi[3]);
  w.kvh = kvh;
  w.row0 = tile * lsh::kTreeRows;
  w.rows = min(lsh::kTreeRows, nodes * a.G - w.row0);
  if (w.seq < 0 || w.seq >= a.S || w.first < 0 || w.first + nodes > a.T || tile < 0 || w.rows <= 0) return false;
  w.rw_bits = w.rows <= kWaveRows ? 0 : (w.rows <= 2 * kWaveRows ? 1 : 2);
  w.tw_bits = 2 - w.rw_bits;
  w.RW = 1 << w.rw_bits;
  w.TW = 1 << w.tw_bits;
  w.rw = wave & (w.RW - 1);
  w.tw = wave >> w.rw_bits;
  w.t0 = max(uniform(lo[2]), 0);
  w.t1 = static_cast<int>(min(static_cast<int64_t>(uniform(lo[3])), static_cast<int64_t>(a.max_blocks) * a.bs));
  return true;
}

// The items [first, last) of a block.
__device__ __forceinline__ void block_items(const TreeArgs& a, int block, int& first, int& last) {
  const int* const starts = a.plan + lsh::plan_starts_at(a.S, a.T, a.items);
  const int blocks = __builtin_amdgcn_readfirstlane(a.plan[0]), items = __builtin_amdgcn_readfirstlane(a.plan[1]);
  first = last = 0;
  if (block >= blocks) return;
  first = max(__builtin_amdgcn_readfirstlane(starts[block]), 0);
  last = min(block + 1 < blocks ? __builtin_amdgcn_readfirstlane(starts[block + 1]) : items, a.items);
}

// This wavefront's tokens for its rows, token after token and row after row in fp32, for ranges with
// cache rows that are not finite: a node that does not see such a row must not be touched by it, and in
// the others an infinity stays in its channel. `put` gets (row of the wavefront, reference, sum, this
// lane's dims lane + 64 i).
template <typename E, int D, int KT, typename Put>
__device__ __forceinline__ void plain_rows(const TreeArgs& a, const Work& w, Put put) {
  constexpr int W = (D + kWave - 1) / kWave;
  const int lane = threadIdx.x % kWave;
  const int64_t* bt = a.bt + static_cast<int64_t>(w.seq) * a.max_blocks;
  const int64_t blocks = a.num_slots / a.bs;
  for (int r = 0; r < kWaveRows; ++r) {
    const int row = w.row0 + kWaveRows * w.rw + r;
    if (row >= w.row0 + w.rows) break;
    const int node = row / a.G, head = w.kvh * a.G + row % a.G;
    const int64_t t = w.first + node;
    const uint64_t see = static_cast<uint64_t>(a.ancestors[t]);
    float q[W], acc[W], m = -1e30f, l = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const int d = lane + kWave * i;
      float v = d < D ? a.q[(t * a.Hq + head) * D + d] : 0.f;
      if (a.q_mult && d < D) v = __fmul_rn(v, a.q_mult[head * D + d]);
      q[i] = v * (a.scale * kLog2e);
      acc[i] = 0.f;
    }
    for (int base = w.t0 + w.tw * KT; base < w.t1; base += w.TW * KT) {
      for (int p = base; p < min(base + KT, w.t1); ++p) {
        if (p >= w.ctx && !(see >> (p - w.ctx) & 1)) continue;
        const int64_t id = bt[p / a.bs];
        if (id < 0 || id >= blocks) continue;
        const int64_t at = (id * a.bs + p % a.bs) * a.Hk + w.kvh;
        float s = 0.f, v[W], ks = 1.f, vs = 1.f;
#pragma unroll
        for (int i = 0; i < W; ++i) {
          const int d = lane + kWave * i;
          v[i] = 0.f;
          if (d < D) {
            s = __builtin_fmaf(q[i], static_cast<float>(static_cast<const E*>(a.kc)[at * D + d]), s);
            v[i] = static_cast<float>(static_cast<const E*>(a.vc)[at * D + d]);
          }
        }
        if constexpr (std::is_same_v<E, int8_t>) {
          ks = a.ks[at];
          vs = a.vs[at];
        }
        s = lsh::group_sum<kWave>(s) * ks;
        const float top = fmaxf(m, s), f = __builtin_amdgcn_exp2f(m - top), e = __builtin_amdgcn_exp2f(s - top);
        m = top;
        l = l * f + e;
#pragma unroll
        for (int i = 0; i < W; ++i) acc[i] = __builtin_fmaf(e * vs, v[i], acc[i] * f);
      }
    }
    put(r, m, l, acc);
  }
}

// What a wavefront has for its rows when its tokens are done.
template <int DT>
struct Rows {
  f32x4 acc[kCols][DT];  // lane (fr, fc): dims DT (4 fc + e) + d of row 16 c + fr
  float ref[kCols], sum[kCols];
  float unscale;         // of acc
  bool bad;              // a cache row was not finite: the rows are computed again by plain_rows
};

// The largest of three. (fmaxf first quiets every operand that came over a branch, an instruction each.)
__device__ __forceinline__ float max3(float x, float y, float z) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "v"(y), "v"(z));
  return r;
}

__device__ __forceinline__ float min3_abs(float x, float y, float z) {
  float r;
  asm("v_min3_f32 %0, |%1|, |%2|, |%3|" : "=v"(r) : "v"(x), "v"(y), "v"(z));
  return r;
}
__device__ __forceinline__ float max3_abs(float x, float y, float z) {
  float r;
  asm("v_max3_f32 %0, |%1|, |%2|, |%3|" : "=v"(r) : "v"(x), "v"(y), "v"(z));
  return r;
}

// From the scores of 32 tokens (lane (fr, fc): tokens 16 tt + 4 fc + e of its rows, in units of 1 / qs) and their V
// scales, the weights times the V scales in two fp16 pieces, in the same lanes; the running reference and
// sum of the rows, and what was summed before, follow. `base`: the first token; `have`: bits of those that are there.
template <int DT>
__device__ __forceinline__ void weights_of(f32x4 (&s)[kCols][2], f32x4 (&vv)[2], const float (&qs)[kCols], const uint64_t (&see)[kCols],
                                           int ctx, int base, uint32_t have, Rows<DT>& o, f16x8 (&ph)[kCols], f16x8 (&pl)[kCols]) {
  constexpr int KT = 32, TT = 2;
  const int fc = threadIdx.x % kWave / 16;
  if (base + KT > ctx || have != 0xffffffffu) {  // tokens of the tree, or some that are not there
    asm volatile("");  // (a branch: as selects for every step it is a fifth of the loop's instructions)
    uint32_t in[kCols];  // bit t: this lane's row sees token t of the step
    const int first = base - ctx;  // the step's first token as a node
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      const uint64_t nodes = first >= 0 ? (first < 64 ? see[c] >> first : 0) : (first > -KT ? see[c] << -first : 0);
      const uint32_t cached = first >= 0 ? 0u : (first > -KT ? (1u << -first) - 1 : 0xffffffffu);
      in[c] = (static_cast<uint32_t>(nodes) | cached) & have;
    }
#pragma unroll
    for (int tt = 0; tt < TT; ++tt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int t = 16 * tt + 4 * fc + e;
        vv[tt][e] = have >> t & 1 ? vv[tt][e] : 0.f;
#pragma unroll
        for (int c = 0; c < kCols; ++c) s[c][tt][e] = in[c] >> t & 1 ? s[c][tt][e] : -__builtin_inff();
      }
  }
  float vtop = max3_abs(vv[0][0], vv[0][1], vv[0][2]);
  vtop = max3_abs(vtop, vv[0][3], vv[1][0]);
  vtop = max3_abs(vtop, vv[1][1], vv[1][2]);
  vtop = max3_abs(vtop, vv[1][3], 0.f);
  float vlow = min3_abs(vv[0][0], vv[0][1], vv[0][2]);
  vlow = min3_abs(vlow, vv[0][3], vv[1][0]);
  vlow = min3_abs(vlow, vv[1][1], vv[1][2]);
  vlow = min3_abs(vlow, vv[1][3], vtop);
  // ---- the running reference: what this lane's weights times V scales stay below, over 2^kTop
  float top[kCols];
  bool raise = false;
  if (__ballot(vlow * 64.f < vtop) == 0) {
    const float lv = fmaxf(__builtin_amdgcn_logf(vtop) - kTop, -kMaxLv);  // the scales' largest will do for all
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      top[c] = max3(s[c][0][0], s[c][0][1], s[c][0][2]);
      top[c] = max3(top[c], s[c][0][3], s[c][1][0]);
      top[c] = max3(top[c], s[c][1][1], s[c][1][2]);
      top[c] = __builtin_fmaf(fmaxf(top[c], s[c][1][3]), qs[c], lv);
    }
  } else {  // a token's own: one of large V and no weight, seen or not, must not push the others out of fp16
    asm volatile("");
#pragma unroll
    for (int c = 0; c < kCols; ++c) top[c] = -__builtin_inff();
#pragma unroll
    for (int tt = 0; tt < TT; ++tt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float lv = fmaxf(__builtin_amdgcn_logf(fabsf(vv[tt][e])) - kTop, -kMaxLv);
#pragma unroll
        for (int c = 0; c < kCols; ++c) top[c] = fmaxf(top[c], __builtin_fmaf(s[c][tt][e], qs[c], lv));
      }
  }
#pragma unroll
  for (int c = 0; c < kCols; ++c) raise |= top[c] > o.ref[c] + kLazy;
  if (__ballot(raise) != 0) {
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      const float want = max_over_fc(top[c]);
      const float now = want > o.ref[c] + kLazy ? want : o.ref[c];
      const float f = __builtin_amdgcn_exp2f(o.ref[c] - now);
      o.ref[c] = now;
      o.sum[c] *= f;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) o.acc[c][d][e] *= f;
    }
  }
  // ---- weights and their product with V
#pragma unroll
  for (int c = 0; c < kCols; ++c) {
    u32x4 hi, lo;
    float eight = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float p[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[c][h][e], qs[c], -o.ref[c]));
        eight += p[e];
      }
      uint32_t h0, l0, h1, l1;
      split2(p[0], vv[h][0], p[1], vv[h][1], h0, l0);
      split2(p[2], vv[h][2], p[3], vv[h][3], h1, l1);
      hi[2 * h] = h0;
      hi[2 * h + 1] = h1;
      lo[2 * h] = l0;
      lo[2 * h + 1] = l1;
    }
    o.sum[c] += eight;
    ph[c] = __builtin_bit_cast(f16x8, hi);
    pl[c] = __builtin_bit_cast(f16x8, lo);
  }
}

template <int D>
constexpr int kMergeRow = D + 4;  // floats of a row in LDS (rows in different banks)

// Joins the wavefronts that share rows, and writes the rows, or their partial results where the sequence
// has several ranges. `acc` [kWaves][kWaveRows][kMergeRow], `rl` [kWaves][kWaveRows][2]; everyone is done with
// what lay there before. The arguments and the work are read again: held since the start, they would be
// spilled around the loop.
template <typename E, int D, int KT>
__device__ __forceinline__ void finish(const TreeArgs& a, const Work& w, Rows<D / 16>& x, float* acc, float* rl, int item) {
  constexpr int DT = D / 16, kRow = kMergeRow<D>;
  int tid = threadIdx.x;
  asm("" : "+v"(tid));  // (what follows from it is formed here, not held since the start)
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave, fr = lane % 16, fc = lane / 16;
  float* const own = acc + wave * kWaveRows * kRow;
  float* const own_rl = rl + wave * kWaveRows * 2;
  if (x.bad) {
    plain_rows<E, D, KT>(a, w, [&](int r, float m, float l, const float (&v)[(D + kWave - 1) / kWave]) {
#pragma unroll
      for (int i = 0; i < D / kWave; ++i) own[r * kRow + lane + kWave * i] = v[i];
      if (lane == 0) {
        own_rl[2 * r] = m;
        own_rl[2 * r + 1] = l;
      }
    });
  } else {
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      const float l = sum_over_fc(x.sum[c]);
      const int r = 16 * c + fr;
      if (fc == 0) {
        own_rl[2 * r] = x.ref[c];
        own_rl[2 * r + 1] = l;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int d = 0; d < DT; d += 4)
          *reinterpret_cast<f32x4*>(own + r * kRow + DT * (4 * fc + e) + d) =
              f32x4{x.acc[c][d][e], x.acc[c][d + 1][e], x.acc[c][d + 2][e], x.acc[c][d + 3][e]} * x.unscale;
    }
  }
  __syncthreads();
  const bool whole = w.ranges <= 1;
  constexpr int LPR = D / 4, kPass = kWaves * kWave / LPR;  // lanes of a row, rows at a time
  const int part = tid % LPR;
  for (int j = tid / LPR; j < w.rows; j += kPass) {
    const int first = j / kWaveRows * kWaveRows + j % kWaveRows, step = w.RW * kWaveRows;  // this row in each share
    float R = -1e30f, L = 0.f;
    for (int k = 0; k < w.TW; ++k) R = fmaxf(R, rl[2 * (first + k * step)]);
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < w.TW; ++k) {
      const int r = first + k * step;
      const float l = rl[2 * r + 1];
      if (l == 0.f) continue;
      const float f = __builtin_amdgcn_exp2f(rl[2 * r] - R);
      L += f * l;
      o += f * *reinterpret_cast<const f32x4*>(acc + r * kRow + 4 * part);
    }
    const int row = w.row0 + j, node = row / a.G, head = w.kvh * a.G + row % a.G;
    if (whole) {
      const float inv = 1.f / L;
      *reinterpret_cast<f32x4*>(a.out + (static_cast<int64_t>(w.first + node) * a.Hq + head) * D + 4 * part) = o * inv;
    } else {
      const int64_t at = (static_cast<int64_t>(item) * a.Hk + w.kvh) * lsh::kTreeRows + j;
      *reinterpret_cast<f32x4*>(a.part_acc + at * D + 4 * part) = o;
      if (part == 0) {
        a.part_rl[2 * at] = R;
        a.part_rl[2 * at + 1] = L;
      }
    }
  }
}

// ---- int8 cache -----------------------------------------------------------------------------------

// Tiles of 32 tokens come straight into LDS as they lie in the cache, a ring of them for each share of the
// tokens: the wavefronts that share a tile bring a part each, one half of the ring while they compute on
// the other. K's 16-byte pieces are permuted within a row, so that 16 tokens' pieces lie in different banks.
// The scores are int8 products: q is scaled to integers of 23 bits, in three signed digits of 8, whose
// products with the codes are summed exactly in 32 bits (K needs no widening). V is widened to fp16.
// An element of q is so held to 2^-24 of its row's largest one: where K's codes in the large channels are near 0, that is what
// a score has left (a channel of q 100 times the others, its K as much smaller: 3e-6 of the result, 1000: 4e-5). A workgroup
// with a row of such elements (kEven) therefore takes q in two fp16 pieces (22 bits of an element down to 2^-29 of the
// largest) and widens K too: 58 us instead of 49 for 16 trees of 26 nodes, 193 instead of 168 for the largest. The test for it
// takes no time that shows.
template <int D>
struct Tile8 {
  static constexpr int KT = 32;
  static constexpr int kSide = KT * D;                // bytes of K, or V
  static constexpr int kBytes = 2 * kSide + KT * 2 * 4;  // and the tokens' K scales, V scales
  static constexpr int kLoads = kSide / 1024;         // 1 KB loads of K, or V
  static constexpr int kChunks = D / 16;              // 16-byte pieces of a row
};
// q as the score products take it.
template <int D>
struct Digits {
  u32x4 d[kCols][D / 64][3];  // the largest last
};
template <int D>
struct Pieces {
  f16x8 hi[kCols][D / 64][2], lo[kCols][D / 64][2];  // lo: times kLoUp
};
// A row takes pieces whose elements' exponents are less than its largest one's by more than this on the mean (normally
// distributed ones' by 2.4, with one of them 16 times as large by 5; an element of 0 counts as one of 1).
constexpr float kEven = 4.5f;
constexpr int kPieceTop = 15;  // a row in pieces has its largest value in [2^14, 2^15)

// A wavefront's rows in pieces: lane (fr, fc) dims fc D / 4 .. + D / 4 of row fr. `qs`: as for digits, for codes times 2^-9.
template <int D>
__device__ __forceinline__ Pieces<D> pieces_of(const TreeArgs& a, const Work& w, int lane, float (&qs)[kCols]) {
  const int fr = lane % 16, fc = lane / 16;
  Pieces<D> q;
#pragma unroll
  for (int c = 0; c < kCols; ++c) {
    const int row = w.row0 + min(kWaveRows * w.rw + 16 * c + fr, w.rows - 1);
    const int node = row / a.G, head = w.kvh * a.G + row % a.G;
    const float* qp = a.q + (static_cast<int64_t>(w.first + node) * a.Hq + head) * D + fc * (D / 4);
    const float* mp = a.q_mult + static_cast<int64_t>(head) * D + fc * (D / 4);
    f32x4 x[D / 16];
    float top = 0.f, odd = 0.f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      x[i] = *reinterpret_cast<const f32x4*>(qp + 4 * i);
      if (a.q_mult) {
        const f32x4 y = *reinterpret_cast<const f32x4*>(mp + 4 * i);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[i][e] = __fmul_rn(x[i][e], y[e]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        top = fmaxf(top, fabsf(x[i][e]));
        odd = __builtin_fmaf(x[i][e], 0.f, odd);
      }
    }
    const int e = kPieceTop - max(__builtin_amdgcn_frexp_expf(max_over_fc(top)), -100);
    const float up = __builtin_copysignf(__builtin_bit_cast(float, static_cast<uint32_t>(127 + e) << 23), a.scale);
    const float down = __builtin_bit_cast(float, static_cast<uint32_t>(127 - e) << 23);
    qs[c] = fmaxf(fabsf(a.scale) * kLog2e * kVUp * down, 1e-37f) + sum_over_fc(odd);
#pragma unroll
    for (int s = 0; s < D / 64; ++s)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        u32x4 hi, lo;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const f32x4 y = x[4 * s + 2 * h + j / 2];
          uint32_t a0, a1;
          split2_up(y[j % 2 * 2], up, y[j % 2 * 2 + 1], up, a0, a1);
          hi[j] = a0;
          lo[j] = a1;
        }
        q.hi[c][s][h] = __builtin_bit_cast(f16x8, hi);
        q.lo[c][s][h] = __builtin_bit_cast(f16x8, lo);
      }
  }
  return q;
}

constexpr int kTiles = 8;                       // of the ring, for all shares together
constexpr int kWindow = 2048, kWindowSlots = kWindow + kWaves * kWave;  // tokens whose slots are looked up at a time
constexpr float kQTop = 8300000.f;              // below 127 * 2^16 + 127 * 2^8 + 127
// An integer below 2^22 added to these bits is that integer plus kMagic as a float: no conversion. The sum of
// the digits' dots carries kMagic along, exact while it is small and one more rounding of 2^-24 when it is not.
constexpr float kMagic = 12582912.f;  // 1.5 * 2^23
constexpr int kMagicBits = 0x4b400000;

// kBytes bytes of each lane to kBytes * lane behind `to` in LDS, past the registers. As the builtin the compiler
// lets every later read of LDS wait for it, which leaves nothing under way while a tile is computed; whoever
// reads the bytes waits for them: vmcnt(0), and a barrier where another wavefront brought them.
template <int kBytes>
__device__ __forceinline__ void load_to_lds(const void* from, char* to) {
  const uint32_t at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)to));
  const uint32_t base = __builtin_amdgcn_readfirstlane(at);
  if constexpr (kBytes == 16)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(base), "v"(from)
                 : "m0", "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(base), "v"(from)
                 : "m0", "memory");
}

struct Room {  // LDS of the workgroup
  char* ring;
  int* slots;
  float* merge_rl;
  int* uneven;  // [kWaves]
};

// An item, with q as Digits, or as Pieces. True: not computed, its q is uneven (the same for the whole workgroup).
template <int D, bool PIECES>
__device__ __forceinline__ bool int8_item(const TreeArgs& a, int item, const Room& room) {
  using T = Tile8<D>;
  constexpr int KT = T::KT, TT = 2, KS = D / 64, DT = D / 16;
  char* const ring = room.ring;
  int* const slots = room.slots;
  int tid = threadIdx.x;
  if constexpr (PIECES) {
    __builtin_amdgcn_s_waitcnt(0x0070);  // the tiles under way have arrived
    __syncthreads();
    asm volatile("" : "+v"(tid)::"memory");  // (formed anew: what both forms shared would be held over the other's loop)
  }
  const int lane = tid % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int fr = lane % 16, fc = lane / 16;
  Work w;
  if (!work_of(a, blockIdx.x, item, wave, w)) return false;
  const int ctx = w.ctx, t1 = w.t1;
  const bool idle = kWaveRows * w.rw >= w.rows;  // no rows: helps to bring tiles

  // ---- the tiles -----------------------------------------------------------------------------------
  const int64_t* bt = a.bt + static_cast<int64_t>(w.seq) * a.max_blocks;
  const int64_t blocks = a.num_slots / a.bs;
  const int64_t stride = static_cast<int64_t>(a.Hk) * D;
  const float* const k_scales = a.ks;  // (a choice between the members would load the pointer per lane)
  const float* const v_scales = a.vs;
  const char* const kc = static_cast<const char*>(a.kc) + w.kvh * D;
  const char* const vc = static_cast<const char*>(a.vc) + w.kvh * D;
  const int depth = kTiles >> w.tw_bits, half = depth / 2;  // tiles of this share's ring
  char* const own_ring = ring + w.tw * depth * T::kBytes;
  auto tile_at = [&](int i) { return own_ring + (i & (depth - 1)) * T::kBytes; };
  // Starts this wavefront's part of the loads of its share's steps [i0, i0 + half) of the window that are below
  // n. A piece is 1 KB of K and the same tokens' of V; there are RW tiles in a half, so every wavefront brings
  // kLoads pieces and a tile's scales.
  const int in_piece = lane / T::kChunks, pos = lane % T::kChunks;  // this lane's token of a piece, and its 16 bytes
  const char* const k_lane = kc + 16 * (pos ^ (in_piece & (T::kChunks - 1)));
  const char* const v_lane = vc + 16 * pos;
  const float* const s_lane = (lane < KT ? k_scales : v_scales) + w.kvh;
  auto issue = [&](int i0, int n) {
    int slot[T::kLoads + 1];
#pragma unroll
    for (int u = 0; u < T::kLoads; ++u) {
      const int id = u << w.rw_bits | w.rw, i = min(i0 + id / T::kLoads, n - 1);
      slot[u] = slots[(i << w.tw_bits | w.tw) * KT + id % T::kLoads * (1024 / D) + in_piece];
    }
    slot[T::kLoads] = slots[(min(i0 + w.rw, n - 1) << w.tw_bits | w.tw) * KT + lane % KT];
#pragma unroll
    for (int u = 0; u < T::kLoads; ++u) {
      const int id = u << w.rw_bits | w.rw, i = i0 + id / T::kLoads;
      if (i >= n) break;
      const int64_t row = max(slot[u], 0) * stride;
      char* const to = tile_at(i) + id % T::kLoads * 1024;
      load_to_lds<16>(k_lane + row, to);
      load_to_lds<16>(v_lane + row, to + T::kSide);
    }
    if (i0 + w.rw < n)
      load_to_lds<4>(s_lane + static_cast<int64_t>(max(slot[T::kLoads], 0)) * a.Hk, tile_at(i0 + w.rw) + 2 * T::kSide);
  };

  // A window's slots: the tables' entries, all reads under way at once, and what becomes of them.
  int64_t ids[kWindowSlots / (kWaves * kWave)];
  auto read_ids = [&](int w0) {
#pragma unroll
    for (int x = 0; x < kWindowSlots / (kWaves * kWave); ++x) {
      const int t = w0 + x * kWaves * kWave + tid;
      ids[x] = -1;
      if (x * kWaves * kWave < kWindow && t < t1) ids[x] = bt[a.bs_shift >= 0 ? t >> a.bs_shift : t / a.bs];
    }
  };
  auto steps_of = [&](int w0) { return ((min(kWindow, t1 - w0) + KT - 1) / KT + w.TW - 1) >> w.tw_bits; };  // of every share
  // writes the slots and starts the loads of the window's first tiles
  auto start_window = [&](int w0) {
    __syncthreads();  // the slots and tiles before it are done with
#pragma unroll
    for (int x = 0; x < kWindowSlots / (kWaves * kWave); ++x) {
      const int at = x * kWaves * kWave + tid, t = w0 + at;
      const int in_block = a.bs_shift >= 0 ? t & (a.bs - 1) : t % a.bs;
      slots[at] = ids[x] >= 0 && ids[x] < blocks ? static_cast<int>(ids[x]) * a.bs + in_block : -1;
    }
    __syncthreads();
    issue(0, steps_of(w0));
  };
  read_ids(w.t0);

  // ---- q: this wavefront's rows as B operands: lane (fr, fc) dims fc D / 4 .. + D / 4 of row fr -------
  uint64_t see[kCols];
  float qs[kCols];  // score = dot * k_scale * qs (log2 units)
#pragma unroll
  for (int c = 0; c < kCols; ++c)
    see[c] = static_cast<uint64_t>(a.ancestors[w.first + (w.row0 + min(kWaveRows * w.rw + 16 * c + fr, w.rows - 1)) / a.G]);
  std::conditional_t<PIECES, Pieces<D>, Digits<D>> q;
  if constexpr (PIECES) {
    start_window(w.t0);
    q = pieces_of<D>(a, w, lane, qs);
  } else {
    // The rows are read in whole lines, 1 KB a load (read as the lanes need them, a lane's row at a time, they
    // took 4 us), and change lanes through the half of the ring that is not under way yet.
    constexpr int LPR = D / 4, kAtOnce = kWave / LPR, kLoads = 16 / kAtOnce;  // lanes of a row, rows of a load
    f32x4 x[kCols][kLoads], mult[kCols][kLoads];
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      const int first = w.row0 + kWaveRows * w.rw + 16 * c, end = w.row0 + w.rows - 1;
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int row = min(first + j * kAtOnce + lane / LPR, end), node = row / a.G, head = w.kvh * a.G + row % a.G;
        x[c][j] = reinterpret_cast<const f32x4*>(a.q + (static_cast<int64_t>(w.first + node) * a.Hq + head) * D)[lane % LPR];
      }
    }
#pragma unroll
    for (int c = 0; c < kCols; ++c)
#pragma unroll
      for (int j = 0; j < kLoads; ++j) mult[c][j] = f32x4{1.f, 1.f, 1.f, 1.f};
    if (a.q_mult) {
#pragma unroll
      for (int c = 0; c < kCols; ++c)
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
          const int row = min(w.row0 + kWaveRows * w.rw + 16 * c + j * kAtOnce + lane / LPR, w.row0 + w.rows - 1);
          const int head = w.kvh * a.G + row % a.G;
          mult[c][j] = reinterpret_cast<const f32x4*>(a.q_mult + static_cast<int64_t>(head) * D)[lane % LPR];
        }
    }

    start_window(w.t0);

    bool uneven = false;  // a row of elements too different in size for digits
    f32x4* const q_lds = reinterpret_cast<f32x4*>(tile_at(half + w.rw));
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      // row r's four dims n at r LPR + (n ^ r): 16 rows' lie in different banks
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int r = j * kAtOnce + lane / LPR;
        q_lds[r * LPR + ((lane % LPR) ^ r)] = x[c][j] * mult[c][j];
      }
      __builtin_amdgcn_wave_barrier();
      float v[D / 4];
      float top = 0.f, odd = 0.f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        const f32x4 y = q_lds[fr * LPR + ((fc * (D / 16) + i) ^ fr)];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[4 * i + e] = y[e];
          top = fmaxf(top, fabsf(y[e]));
          odd = __builtin_fmaf(y[e], 0.f, odd);  // NaN where q is not finite
        }
      }
      __builtin_amdgcn_wave_barrier();
      top = max_over_fc(top);
      odd = sum_over_fc(odd);
      int bits = 0;  // of the elements' exponents
#pragma unroll
      for (int i = 0; i < D / 4; ++i) bits += __builtin_amdgcn_frexp_expf(v[i]);
      uneven |= __ballot(D * __builtin_amdgcn_frexp_expf(top) - sum_over_fc(static_cast<float>(bits)) > kEven * D) != 0;
      const float f = fminf(kQTop / top, 1e37f);  // (0: 1e37)
      // the sign of the softmax scale goes with q, so that the scores' order is the dots'; qs > 0: -inf * 0 below
      const float up = __builtin_copysignf(f, a.scale);
      qs[c] = fmaxf(fabsf(a.scale) * kLog2e / f, 1e-37f) + odd;
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // n + 0x808080 has the digits, each plus 128, as its bytes: the bytes of four elements transposed
          uint32_t m[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            m[e] = static_cast<uint32_t>(static_cast<int>(__builtin_rintf(v[16 * s + 4 * i + e] * up)) + 0x808080);
          const uint32_t p01 = __builtin_amdgcn_perm(m[1], m[0], 0x05010400u), p23 = __builtin_amdgcn_perm(m[3], m[2], 0x05010400u);
          const uint32_t h01 = __builtin_amdgcn_perm(m[1], m[0], 0x07030602u), h23 = __builtin_amdgcn_perm(m[3], m[2], 0x07030602u);
          const uint32_t digit[3] = {__builtin_amdgcn_perm(p23, p01, 0x05040100u) ^ 0x80808080u,
                                     __builtin_amdgcn_perm(p23, p01, 0x07060302u) ^ 0x80808080u,
                                     __builtin_amdgcn_perm(h23, h01, 0x05040100u) ^ 0x80808080u};
#pragma unroll
          for (int g = 0; g < 3; ++g) q.d[c][s][g][i] = digit[g];
        }
    }
    if (w.RW > 1) {  // the same for the whole workgroup (without row groups all have the same rows)
      if (lane == 0) room.uneven[wave] = uneven;
      __syncthreads();
      uneven = __builtin_amdgcn_readfirstlane(room.uneven[0] | room.uneven[1] | room.uneven[2] | room.uneven[3]) != 0;
    }
    if (uneven) return true;
  }

  Rows<DT> o;
#pragma unroll
  for (int c = 0; c < kCols; ++c) {
    o.ref[c] = -1e30f;
    o.sum[c] = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) o.acc[c][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  o.bad = false;

  auto compute = [&](int i, int base) {
    const char* const tile = tile_at(i);
    const float* const scales = reinterpret_cast<const float*>(tile + 2 * T::kSide);
    const uint32_t have = static_cast<uint32_t>(__ballot(slots[(i << w.tw_bits | w.tw) * KT + lane % KT] >= 0));
    const float mine = scales[lane];
    // a scale that is not finite, or one too large to stage
    o.bad |= __ballot((have >> (lane % KT) & 1) && !(fabsf(mine) < 1e30f)) != 0;
    // ---- what the scores need of the tile, before the first product waits for any of it
    i32x4 k[TT][KS];
    f32x4 s[kCols][TT], kk[TT], vv[TT];
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int row = 16 * tt + fr, chunk = (fc * KS + ks) ^ (row & (T::kChunks - 1));
        k[tt][ks] = *reinterpret_cast<const i32x4*>(tile + row * D + 16 * chunk);
      }
      kk[tt] = *reinterpret_cast<const f32x4*>(scales + 16 * tt + 4 * fc);
      vv[tt] = *reinterpret_cast<const f32x4*>(scales + KT + 16 * tt + 4 * fc);
    }
    __builtin_amdgcn_sched_barrier(0);
    // ---- scores: lane (fr, fc) gets tokens 16 tt + 4 fc + e of its rows
    if constexpr (!PIECES) {
#pragma unroll
      for (int tt = 0; tt < TT; ++tt) {
        const f32x4 kk_magic = kk[tt] * kMagic;
        i32x4 dot[kCols][3] = {};
#pragma unroll
        for (int c = 0; c < kCols; ++c) dot[c][0] = i32x4{kMagicBits, kMagicBits, kMagicBits, kMagicBits};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
          for (int g = 0; g < 3; ++g)
#pragma unroll
            for (int c = 0; c < kCols; ++c)
              dot[c][g] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k[tt][ks], __builtin_bit_cast(i32x4, q.d[c][ks][g]), dot[c][g], 0, 0, 0);
        }
#pragma unroll
        for (int c = 0; c < kCols; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int high = (dot[c][2][e] << 8) + dot[c][1][e], low = dot[c][0][e];
            s[c][tt][e] = __builtin_fmaf(__builtin_fmaf(static_cast<float>(high), 256.f, __builtin_bit_cast(float, low)),
                                         kk[tt][e], -kk_magic[e]);
          }
      }
    } else {
#pragma unroll
      for (int tt = 0; tt < TT; ++tt) {
        f32x4 high[kCols] = {}, low[kCols] = {};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const u32x2 x = codes_to_h2(static_cast<uint32_t>(k[tt][ks][2 * h])), y = codes_to_h2(static_cast<uint32_t>(k[tt][ks][2 * h + 1]));
            const f16x8 kf = __builtin_bit_cast(f16x8, u32x4{x[0], x[1], y[0], y[1]});
#pragma unroll
            for (int c = 0; c < kCols; ++c) low[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, q.lo[c][ks][h], low[c], 0, 0, 0);
#pragma unroll
            for (int c = 0; c < kCols; ++c) high[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, q.hi[c][ks][h], high[c], 0, 0, 0);
          }
#pragma unroll
        for (int c = 0; c < kCols; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[c][tt][e] = __builtin_fmaf(low[c][e], 1.f / kLoUp, high[c][e]) * kk[tt][e];
      }
    }
    uint32_t y[8][D / 64];  // V: dims fr D / 16 .. of tokens 4 fc + e and 16 + 4 fc + e
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const char* p = tile + T::kSide + fr * DT + (16 * (e / 4) + 4 * fc + e % 4) * D;
      if constexpr (D == 128) {
        const u32x2 x = *reinterpret_cast<const u32x2*>(p);
        y[e][0] = x[0];
        y[e][1] = x[1];
      } else {
        y[e][0] = *reinterpret_cast<const uint32_t*>(p);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    f16x8 ph[kCols], pl[kCols];
    weights_of<DT>(s, vv, qs, see, ctx, base, have, o, ph, pl);
#pragma unroll
    for (int g = 0; g < D / 64; ++g) {  // four dims of 8 tokens
      uint32_t x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = y[e][g] ^ 0x80808080u;
#pragma unroll
      for (int j0 = 0; j0 < 4; j0 += 2) {  // (four sums, so that a product does not wait for the one before)
        f16x8 vf[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          u32x4 v;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            v[e] = j0 + j == 0   ? bytes_to_h2<0>(x[2 * e], x[2 * e + 1])
                   : j0 + j == 1 ? bytes_to_h2<1>(x[2 * e], x[2 * e + 1])
                   : j0 + j == 2 ? bytes_to_h2<2>(x[2 * e], x[2 * e + 1])
                                 : bytes_to_h2<3>(x[2 * e], x[2 * e + 1]);
          vf[j] = __builtin_bit_cast(f16x8, v);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int c = 0; c < kCols; ++c)
              o.acc[c][4 * g + j0 + j] =
                  __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[j], h == 0 ? pl[c] : ph[c], o.acc[c][4 * g + j0 + j], 0, 0, 0);
      }
    }
  };

  for (int w0 = w.t0; w0 < t1; w0 += kWindow) {
    if (w0 != w.t0) {
      read_ids(w0);
      start_window(w0);
    }
    const int n = steps_of(w0);
    for (int i0 = 0; i0 < n; i0 += half) {
      // this wavefront's part is there, and it has read the other half; after the barrier both hold for all
      __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
      if (w.RW > 1) __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (i0 + half < n) issue(i0 + half, n);
      if (idle) continue;
      for (int i = i0; i < min(i0 + half, n); ++i) compute(i, w0 + (i << w.tw_bits | w.tw) * KT);
    }
  }
  __syncthreads();
  o.unscale = kVUp;
  finish<int8_t, D, KT>(a, w, o, reinterpret_cast<float*>(ring), room.merge_rl, item);
  return false;
}

template <int D>
__global__ __launch_bounds__(kWaves* kWave, 2) void tree_int8_kernel(TreeArgs a) {
  using T = Tile8<D>;
  constexpr int kMerge = kWaves * kWaveRows * kMergeRow<D> * 4;  // the ring holds the results in the end
  __shared__ __attribute__((aligned(16))) char ring[kTiles * T::kBytes > kMerge ? kTiles * T::kBytes : kMerge];
  __shared__ int slots[kWindowSlots];
  __shared__ float merge_rl[kWaves * kWaveRows * 2];
  __shared__ int uneven[kWaves];
  const Room room{ring, slots, merge_rl, uneven};
  int first, last;
  block_items(a, blockIdx.y, first, last);
  // The items with uneven q come after the others: in one loop, what the two forms hold is spilled (56 us for 16 trees, in
  // loops of their own 49). Bits of the items; those past the 31st share one, and are all computed (again) in pieces.
  uint32_t todo = 0;
  for (int item = first; item < last; ++item)
    if (int8_item<D, false>(a, item, room)) todo |= 1u << min(item - first, 31);
  todo = __builtin_amdgcn_readfirstlane(todo);
  for (; todo; todo &= todo - 1) {
    const int i = __builtin_ctz(todo);
    for (int item = first + i; item < (i < 31 ? first + i + 1 : last); ++item) int8_item<D, true>(a, item, room);
  }
}

// ---- fp32 cache -----------------------------------------------------------------------------------

// Trees of many rows: fp16 matrix instructions on K, V, q and weights in two fp16 pieces, three products
// for each (the low pieces' own is below the last bit). A row of K, V or q is scaled by a power of two (largest value in
// [2^14, 2^15)), its low pieces by 2^11 more: an element keeps 22 bits down to 2^-29 of its row's largest, and is held to
// 2^-51 of that below. (With the low pieces as they come and V in [2^4, 2^5), one channel 10^4 times the others left
// those 8e-6; the scaling takes 1 us of 45.) The low pieces' products with q have sums of their own, those with the
// weights take high pieces of 2^-11. All wavefronts take the same 32 tokens: each brings and splits a quarter of
// them, two tokens and 8 dims a lane, into one half of LDS while the other is computed; V is laid down
// with the tokens of a product step side by side, so that no wavefront transposes. Addresses in the loop are formed
// anew for every tile: kept, they were spilled, and reading them back waits for the rows under way (57 us instead
// of 47). Rows that are not finite leave NaN in the sums, and plain_rows takes over.
constexpr float kVPieceUp = 1024.f;      // of that, what the weights do not take back (p v_scale lies near 2^kTop with V near 2^5)
template <int D>
__global__ __launch_bounds__(kWaves* kWave, 2) void tree_split_kernel(TreeArgs a) {
  constexpr int KT = 32, KS = D / 32, DT = D / 16, kSide = KT * D * 2, kRowBytes = 4 * D, kHalf = 4 * kSide + 2 * KT * 4;
  static_assert(D == 128, "a thread stages two tokens' 8 dims");
  constexpr int kMerge = kWaves * kWaveRows * kMergeRow<D> * 4;  // the results lie there in the end
  __shared__ __attribute__((aligned(16))) char lds[2 * kHalf > kMerge ? 2 * kHalf : kMerge];
  __shared__ float merge_rl[kWaves * kWaveRows * 2];
  const int tid = threadIdx.x, lane = tid % kWave, fr = lane % 16, fc = lane / 16;
  int item, last;
  block_items(a, blockIdx.y, item, last);
  for (; item < last; ++item) {
  Work w;
  if (!work_of(a, blockIdx.x, item, 0, w)) continue;
  __syncthreads();  // the last item's rows have been read from LDS
  w.rw = __builtin_amdgcn_readfirstlane(tid / kWave);
  w.RW = kWaves;
  w.tw = 0;
  w.TW = 1;
  const int ctx = w.ctx, t1 = w.t1, n = t1 > w.t0 ? (t1 - w.t0 + KT - 1) / KT : 0;
  const bool idle = kWaveRows * w.rw >= w.rows;

  // ---- the tokens: lane's tokens 2 (tid / 16) + k of a tile, dims 8 (tid % 16) .. + 8 --------------
  const int64_t* bt = a.bt + static_cast<int64_t>(w.seq) * a.max_blocks;
  const int64_t blocks = a.num_slots / a.bs;
  const int64_t stride = static_cast<int64_t>(a.Hk) * kRowBytes;
  const char* const kc = static_cast<const char*>(a.kc) + w.kvh * kRowBytes;
  const char* const vc = static_cast<const char*>(a.vc) + w.kvh * kRowBytes;
  auto my_tid = [] {  // (what follows from it is formed at its use: held, it is spilled, and its reload waits for the loads)
    int tid = threadIdx.x;
    asm("" : "+v"(tid));
    return tid;
  };
  auto block_of = [&](int t) { return a.bs_shift >= 0 ? t >> a.bs_shift : t / a.bs; };
  int64_t id[2];
  auto fetch = [&](int i) {
    const int mine = my_tid() / 16 * 2;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int t = w.t0 + i * KT + mine + k;
      id[k] = t < t1 ? bt[block_of(t)] : static_cast<int64_t>(-1);
    }
  };
  f32x4 kx[2][2], vx[2][2];
  bool on[2];
  auto load = [&](int i) {
    const int tid = my_tid(), mine = tid / 16 * 2, chunk = tid % 16;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int t = w.t0 + i * KT + mine + k;
      on[k] = id[k] >= 0 && id[k] < blocks;
      const int64_t row = (on[k] ? static_cast<int>(id[k]) * a.bs + (t - block_of(t) * a.bs) : 0) * stride + 32 * chunk;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        kx[k][h] = *reinterpret_cast<const f32x4*>(kc + row + 16 * h);
        vx[k][h] = *reinterpret_cast<const f32x4*>(vc + row + 16 * h);
      }
    }
  };
  // 2^(to - exponent of the row's largest value) and its inverse; 16 lanes have the row
  auto scale_of = [](const f32x4 (&x)[2], int to, float& up, float& down) {
    float m = max3_abs(x[0][0], x[0][1], x[0][2]);
    m = max3_abs(m, x[0][3], x[1][0]);
    m = max3_abs(m, x[1][1], x[1][2]);
    m = max3_abs(m, x[1][3], 0.f);
    m = fmaxf(m, row_lane<0xb1>(m));   // lanes ^ 1
    m = fmaxf(m, row_lane<0x4e>(m));   // lanes ^ 2
    m = fmaxf(m, row_lane<0x141>(m));  // 8 lanes mirrored
    m = fmaxf(m, row_lane<0x140>(m));  // 16 lanes mirrored
    // (a row of zeros must not count as one of large values)
    const int e = to - (m > 0.f ? max(__builtin_amdgcn_frexp_expf(m), -100) : -100);
    up = __builtin_bit_cast(float, static_cast<uint32_t>(127 + e) << 23);
    down = __builtin_bit_cast(float, static_cast<uint32_t>(127 - e) << 23);
  };
  auto stage = [&](char* to) {
    const int tid = my_tid(), mine = tid / 16 * 2, chunk = tid % 16;
    const int place = mine % 16 / 4 * 8 + mine / 16 * 4 + mine % 4;  // of the first token among a V row's
    if (__ballot(!on[0] || !on[1]) != 0) {  // (a row that is not there may hold anything)
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          kx[k][h] = on[k] ? kx[k][h] : f32x4{0.f, 0.f, 0.f, 0.f};
          vx[k][h] = on[k] ? vx[k][h] : f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }
    float* const scales = reinterpret_cast<float*>(to + 4 * kSide);
    float up[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float each, down;
      scale_of(kx[k], kPieceTop, each, down);
      u32x4 hi, lo;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t h, l;
        split2_up(kx[k][j / 2][j % 2 * 2], each, kx[k][j / 2][j % 2 * 2 + 1], each, h, l);
        hi[j] = h;
        lo[j] = l;
      }
      const int row = mine + k, at = row * 2 * D + 16 * (chunk ^ (row & 15));
      *reinterpret_cast<u32x4*>(to + at) = hi;
      *reinterpret_cast<u32x4*>(to + kSide + at) = lo;
      if (chunk == 0) scales[row] = on[k] ? down : 0.f;
      scale_of(vx[k], kPieceTop, up[k], down);
      if (chunk == 0) scales[KT + row] = on[k] ? down * kVPieceUp : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {  // dim 8 chunk + j: row chunk of product j
      uint32_t h, l;
      split2_up(vx[0][j / 4][j % 4], up[0], vx[1][j / 4][j % 4], up[1], h, l);
      const int at = (j * 16 + chunk) * 64 + 16 * ((place / 8) ^ (chunk / 4)) + place % 8 * 2;
      *reinterpret_cast<uint32_t*>(to + 2 * kSide + at) = h;
      *reinterpret_cast<uint32_t*>(to + 3 * kSide + at) = l;
    }
  };
  // ---- q: this wavefront's rows as B operands: lane (fr, fc) dims 32 ks + 8 fc .. + 8 of row fr; read
  // before the first tokens' rows, split while those are under way
  uint64_t see[kCols];
  float qs[kCols];
  f16x8 qh[kCols][KS], ql[kCols][KS];
  f32x4 x[kCols][KS][2];
  fetch(0);
#pragma unroll
  for (int c = 0; c < kCols; ++c) {
    const int row = w.row0 + min(kWaveRows * w.rw + 16 * c + fr, w.rows - 1);
    const int node = row / a.G, head = w.kvh * a.G + row % a.G;
    see[c] = static_cast<uint64_t>(a.ancestors[w.first + node]);
    const float* qp = a.q + (static_cast<int64_t>(w.first + node) * a.Hq + head) * D + 8 * fc;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int h = 0; h < 2; ++h) x[c][ks][h] = *reinterpret_cast<const f32x4*>(qp + 32 * ks + 4 * h);
  }
  load(0);
  fetch(1);
  if (a.q_mult) {
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      const int row = w.row0 + min(kWaveRows * w.rw + 16 * c + fr, w.rows - 1);
      const float* mp = a.q_mult + static_cast<int64_t>(w.kvh * a.G + row % a.G) * D + 8 * fc;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const f32x4 y = *reinterpret_cast<const f32x4*>(mp + 32 * ks + 4 * h);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[c][ks][h][e] = __fmul_rn(x[c][ks][h][e], y[e]);
        }
    }
  }
#pragma unroll
  for (int c = 0; c < kCols; ++c) {
    float top = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        top = max3_abs(top, x[c][ks][h][0], x[c][ks][h][1]);
        top = max3_abs(top, x[c][ks][h][2], x[c][ks][h][3]);
      }
    const int e = kPieceTop - max(__builtin_amdgcn_frexp_expf(max_over_fc(top)), -100);
    // the sign of the softmax scale goes with q, so that the scores' order is the dots'; qs > 0: -inf * 0 below
    const float up = __builtin_copysignf(__builtin_bit_cast(float, static_cast<uint32_t>(127 + e) << 23), a.scale);
    qs[c] = fmaxf(fabsf(a.scale) * kLog2e * __builtin_bit_cast(float, static_cast<uint32_t>(127 - e) << 23), 1e-37f);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      u32x4 hi, lo;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t h, l;
        split2_up(x[c][ks][j / 2][j % 2 * 2], up, x[c][ks][j / 2][j % 2 * 2 + 1], up, h, l);
        hi[j] = h;
        lo[j] = l;
      }
      qh[c][ks] = __builtin_bit_cast(f16x8, hi);
      ql[c][ks] = __builtin_bit_cast(f16x8, lo);
    }
  }
  Rows<DT> o;
#pragma unroll
  for (int c = 0; c < kCols; ++c) {
    o.ref[c] = -1e30f;
    o.sum[c] = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) o.acc[c][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  auto compute = [&](const char* tile, int base) {
    const int lane = my_tid() % kWave, fr = lane % 16, fc = lane / 16;
    const float* const scales = reinterpret_cast<const float*>(tile + 4 * kSide);
    const uint32_t have = static_cast<uint32_t>(__ballot(scales[lane % KT] != 0.f));
    f32x4 s[kCols][2], vv[2];
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
      // (four sums, so that a product does not wait for the one before; the low pieces' in their own, kLoUp as large)
      f32x4 high[kCols] = {}, low[kCols] = {};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const char* p = tile + (16 * tt + fr) * 2 * D + 16 * ((4 * ks + fc) ^ fr);
        const f16x8 kh = *reinterpret_cast<const f16x8*>(p), kl = *reinterpret_cast<const f16x8*>(p + kSide);
#pragma unroll
        for (int c = 0; c < kCols; ++c) low[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kl, qh[c][ks], low[c], 0, 0, 0);
#pragma unroll
        for (int c = 0; c < kCols; ++c) high[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, qh[c][ks], high[c], 0, 0, 0);
#pragma unroll
        for (int c = 0; c < kCols; ++c) low[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, ql[c][ks], low[c], 0, 0, 0);
      }
      const f32x4 kk = *reinterpret_cast<const f32x4*>(scales + 16 * tt + 4 * fc);
      vv[tt] = *reinterpret_cast<const f32x4*>(scales + KT + 16 * tt + 4 * fc);
#pragma unroll
      for (int c = 0; c < kCols; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[c][tt][e] = __builtin_fmaf(low[c][e], 1.f / kLoUp, high[c][e]) * kk[e];
    }
    f16x8 ph[kCols], pl[kCols], pd[kCols];  // pd: for V's low pieces
    weights_of<DT>(s, vv, qs, see, ctx, base, have, o, ph, pl);
#pragma unroll
    for (int c = 0; c < kCols; ++c) pd[c] = ph[c] * static_cast<_Float16>(1.f / kLoUp);
#pragma unroll
    for (int d0 = 0; d0 < DT; d0 += 2) {
      f16x8 vh[2], vl[2];
#pragma unroll
      for (int d = 0; d < 2; ++d) {
        const char* p = tile + 2 * kSide + ((d0 + d) * 16 + fr) * 64 + 16 * (fc ^ (fr / 4));
        vh[d] = *reinterpret_cast<const f16x8*>(p);
        vl[d] = *reinterpret_cast<const f16x8*>(p + kSide);
      }
#pragma unroll
      for (int g = 0; g < 3; ++g)
#pragma unroll
        for (int d = 0; d < 2; ++d)
#pragma unroll
          for (int c = 0; c < kCols; ++c)
            o.acc[c][d0 + d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(g == 0 ? vl[d] : vh[d], g == 0 ? pd[c] : g == 1 ? pl[c] : ph[c], o.acc[c][d0 + d], 0, 0, 0);
    }
  };
  // everyone's part of the next tile is there, and this one has been read; loads stay under way
  auto meet = [] {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  if (n > 0) stage(lds);
  if (n > 1) load(1);
  fetch(2);
  meet();
  for (int i = 0; i < n; ++i) {
    if (!idle) compute(lds + (i & 1) * kHalf, w.t0 + i * KT);
    if (i + 1 < n) {
      stage(lds + (~i & 1) * kHalf);
      if (i + 2 < n) load(i + 2);
      fetch(i + 3);
    }
    meet();
  }
  o.unscale = 1.f / kVPieceUp;
  float odd = 0.f;  // NaN where a sum is not finite
#pragma unroll
  for (int c = 0; c < kCols; ++c) {
    odd = __builtin_fmaf(o.sum[c], 0.f, odd);
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) odd = __builtin_fmaf(o.acc[c][d][e], 0.f, odd);
  }
  o.bad = __ballot(odd != odd) != 0;
  finish<float, D, KT>(a, w, o, reinterpret_cast<float*>(lds), merge_rl, item);
  }
}

// Steps of 16 tokens, on the fp32 matrix instructions. A wavefront reads its tokens from the cache into
// registers: the next step's K as soon as this step's scores are formed, its V when the products with this
// step's are issued.
template <int D>
__global__ __launch_bounds__(kWaves* kWave, 2) void tree_f32_kernel(TreeArgs a) {
  constexpr int KT = 16, DT = D / 16, kRowBytes = 4 * D;
  constexpr uint32_t kAll = (1u << KT) - 1;
  __shared__ __attribute__((aligned(16))) float merge_acc[kWaves * kWaveRows * kMergeRow<D>];
  __shared__ float merge_rl[kWaves * kWaveRows * 2];
  __shared__ __attribute__((aligned(16))) int64_t offsets[kWaves][KT];  // of the step's rows in a cache, bytes

  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
  const int fr = lane % 16, fc = lane / 16;
  int item, last;
  block_items(a, blockIdx.y, item, last);
  for (; item < last; ++item) {
  Work w;
  if (!work_of(a, blockIdx.x, item, wave, w)) continue;
  const int ctx = w.ctx, t1 = w.t1;
  __syncthreads();  // the last item's rows have been read from LDS
  // ---- q: this wavefront's rows as B operands, waiting in the part of LDS that its results take later --
  uint64_t see[kCols];
  f32x4* const q_lds = reinterpret_cast<f32x4*>(merge_acc + wave * kWaveRows * kMergeRow<D>) + lane;
  // score = dot * qs (log2 units); the sign of the softmax scale goes with q, so that the scores' order is
  // the dots' (and qs > 0: -inf * 0 below)
  const float qs = fmaxf(fabsf(a.scale) * kLog2e, 1e-37f);
#pragma unroll
  for (int c = 0; c < kCols; ++c) {
    const int row = w.row0 + min(kWaveRows * w.rw + 16 * c + fr, w.rows - 1);
    const int node = row / a.G, head = w.kvh * a.G + row % a.G;
    see[c] = static_cast<uint64_t>(a.ancestors[w.first + node]);
    const float* qp = a.q + (static_cast<int64_t>(w.first + node) * a.Hq + head) * D + fc * (D / 4);
    const float* mp = a.q_mult + static_cast<int64_t>(head) * D + fc * (D / 4);
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      f32x4 x = *reinterpret_cast<const f32x4*>(qp + 4 * i);
      if (a.q_mult) {
        const f32x4 y = *reinterpret_cast<const f32x4*>(mp + 4 * i);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = __fmul_rn(x[e], y[e]);
      }
      q_lds[(c * (D / 16) + i) * kWave] = a.scale < 0.f ? -x : x;
    }
  }

  // ---- the tokens: block ids two steps ahead, rows ahead of their use ------------------------------
  const int64_t* bt = a.bt + static_cast<int64_t>(w.seq) * a.max_blocks;
  const int64_t blocks = a.num_slots / a.bs;
  const int64_t stride = static_cast<int64_t>(a.Hk) * kRowBytes;
  const char* const k_lane = static_cast<const char*>(a.kc) + w.kvh * kRowBytes + fc * (kRowBytes / 4);
  const char* const v_lane = static_cast<const char*>(a.vc) + w.kvh * kRowBytes + fr * (kRowBytes / 16);
  auto base_of = [&](int i) { return w.t0 + (w.tw + i * w.TW) * KT; };  // first token of this wavefront's step i
  auto block_of = [&](int t) { return a.bs_shift >= 0 ? t >> a.bs_shift : t / a.bs; };
  auto fetch_id = [&](int i) {
    const int t = base_of(i) + lane % KT;
    return t < t1 ? bt[block_of(t)] : static_cast<int64_t>(-1);
  };
  f32x4 k[D / 16];     // token fr, dims fc D / 4 .. + D / 4
  f32x4 v[4][D / 64];  // tokens 4 fc + e, dims fr D / 16 .. + D / 16
  uint32_t have = 0, next_have = 0;  // bits: the step's tokens that are there
  auto load_k = [&](int i, int64_t id) {
    const int t = base_of(i) + lane % KT;
    const int slot = id < 0 || id >= blocks ? -1 : static_cast<int>(id) * a.bs + (t - block_of(t) * a.bs);
    next_have = static_cast<uint32_t>(__ballot(slot >= 0)) & kAll;
    if (lane < KT) offsets[wave][lane] = max(slot, 0) * stride;
    __builtin_amdgcn_wave_barrier();
    const char* p = k_lane + offsets[wave][fr];
#pragma unroll
    for (int j = 0; j < D / 16; ++j) k[j] = *reinterpret_cast<const f32x4*>(p + 16 * j);
  };
  auto load_v = [&] {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const char* p = v_lane + offsets[wave][4 * fc + e];
#pragma unroll
      for (int j = 0; j < D / 64; ++j) v[e][j] = *reinterpret_cast<const f32x4*>(p + 16 * j);
    }
    __builtin_amdgcn_wave_barrier();
  };

  // this wavefront's steps: tw, tw + TW, ... of the range's; none where it has no rows
  const int n = w.t0 + w.tw * KT < t1 && kWaveRows * w.rw < w.rows ? (t1 - w.t0 - w.tw * KT + w.TW * KT - 1) / (w.TW * KT) : 0;
  int64_t id = fetch_id(0);
  if (n > 0) {
    load_k(0, id);
    load_v();
  }
  have = next_have;
  id = fetch_id(1);

  Rows<DT> o;
#pragma unroll
  for (int c = 0; c < kCols; ++c) {
    o.ref[c] = -1e30f;
    o.sum[c] = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) o.acc[c][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  o.bad = false;  // a tree's cache row that is not finite (a cached one is seen by all rows)

  for (int i = 0; i < n; ++i) {
    const int base = base_of(i);
    // ---- scores: lane (fr, fc) gets tokens 4 fc + e of its rows
    f32x4 s[kCols];
    {
      f32x4 part[kCols][2] = {};
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        f32x4 q[kCols];
#pragma unroll
        for (int c = 0; c < kCols; ++c) q[c] = q_lds[(c * (D / 16) + j) * kWave];
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int c = 0; c < kCols; ++c)
            part[c][e % 2] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[j][e], q[c][e], part[c][e % 2], 0, 0, 0);
      }
#pragma unroll
      for (int c = 0; c < kCols; ++c) s[c] = part[c][0] + part[c][1];
    }
    {  // (past the last step: slot 0, not there)
      const int64_t now = id;
      id = fetch_id(i + 2);
      load_k(i + 1, now);
    }
    if (base + KT > ctx || have != kAll) {  // tokens of the tree, or some that are not there
      uint32_t in[kCols];  // bit t: this lane's row sees token t of the step
      const int first = base - ctx;  // the step's first token as a node
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        const uint64_t nodes = first >= 0 ? (first < 64 ? see[c] >> first : 0) : (first > -KT ? see[c] << -first : 0);
        const uint32_t cached = first >= 0 ? 0u : (first > -KT ? (1u << -first) - 1 : kAll);
        in[c] = (static_cast<uint32_t>(nodes) | cached) & have;
      }
      bool odd = false;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
#pragma unroll
        for (int c = 0; c < kCols; ++c) s[c][e] = in[c] >> (4 * fc + e) & 1 ? s[c][e] : -__builtin_inff();
#pragma unroll
        for (int j = 0; j < D / 64; ++j)
#pragma unroll
          for (int d = 0; d < 4; ++d) {
            const float x = have >> (4 * fc + e) & 1 ? v[e][j][d] : 0.f;
            v[e][j][d] = x;
            odd |= !(fabsf(x) < __builtin_inff());
          }
      }
      o.bad |= __ballot(odd) != 0;
    }
    // ---- the running reference
    float top[kCols];
    bool raise = false;
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      top[c] = fmaxf(fmaxf(s[c][0], s[c][1]), fmaxf(s[c][2], s[c][3])) * qs;
      raise |= top[c] > o.ref[c] + kLazy;
    }
    if (__ballot(raise) != 0) {
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        const float want = max_over_fc(top[c]);
        const float now = want > o.ref[c] + kLazy ? want : o.ref[c];
        const float f = __builtin_amdgcn_exp2f(o.ref[c] - now);
        o.ref[c] = now;
        o.sum[c] *= f;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e) o.acc[c][d][e] *= f;
      }
    }
    // ---- weights and their product with V: the step's sum apart, one rounding at acc's size
    float p[kCols][4];
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      float four = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        p[c][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[c][e], qs, -o.ref[c]));
        four += p[c][e];
      }
      o.sum[c] += four;
    }
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      f32x4 t[kCols] = {};
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int c = 0; c < kCols; ++c)
          t[c] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[e][d / 4][d % 4], p[c][e], t[c], 0, 0, 0);
#pragma unroll
      for (int c = 0; c < kCols; ++c) o.acc[c][d] += t[c];
    }
    load_v();
    have = next_have;
  }
  o.unscale = 1.f;
  __syncthreads();
  finish<float, D, KT>(a, w, o, merge_acc, merge_rl, item);
  }
}

// Adds the ranges of the sequences that have several: D / 4 lanes per row.
//   R = max_j r_j;  out = sum_j 2^(r_j - R) acc_j / sum_j 2^(r_j - R) l_j   (l_j = 0 skipped)
template <int D>
__global__ __launch_bounds__(kWaves* kWave) void tree_merge_kernel(TreeArgs a) {
  constexpr int LPR = D / 4, kBatch = 4;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * (kWaves * kWave / LPR) + threadIdx.x / LPR;
  const int part = threadIdx.x % LPR;
  if (i >= a.T * a.Hq) return;
  const int64_t t = i / a.Hq;
  const int head = static_cast<int>(i % a.Hq);
  const int seq = a.plan[lsh::plan_owners_at(a.S) + t];
  if (seq < 0 || seq >= a.S) return;
  const DraftSeq u = lsh::plan_seqs(a.plan)[seq];
  const int kvh = head / a.G;
  const int64_t row = (t - u.first) * a.G + head % a.G, Q = a.plan[2];
  const int64_t cost = a.plan[3];
  if (row < 0 || Q <= 0 || u.off < 0 || u.len <= 0) return;
  int64_t first = u.item0, off = u.off;
  for (int r = 0; r < row / lsh::kTreeRows; ++r) {
    first += lsh::cut_tile(off, u.len, Q, cost).items;
    off = (off + lsh::tile_span(u.len, Q, cost)) % Q;
  }
  const int n = static_cast<int>(lsh::cut_tile(off, u.len, Q, cost).items);
  if (n <= 1 || first < 0 || first + n > a.items) return;
  float R = -1e30f, L = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int j0 = 0; j0 < n; j0 += kBatch) {
    float r[kBatch], l[kBatch];
    f32x4 v[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int64_t at = ((first + min(j0 + j, n - 1)) * a.Hk + kvh) * lsh::kTreeRows + row % lsh::kTreeRows;
      r[j] = a.part_rl[2 * at];
      l[j] = a.part_rl[2 * at + 1];
      v[j] = *reinterpret_cast<const f32x4*>(a.part_acc + at * D + 4 * part);
    }
    float top = R;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) top = fmaxf(top, r[j]);
    const float f = __builtin_amdgcn_exp2f(R - top);
    R = top;
    L *= f;
    o *= f;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const bool on = j0 + j < n && l[j] != 0.f;
      const float wt = on ? __builtin_amdgcn_exp2f(r[j] - R) : 0.f;
      L += wt * l[j];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += wt * (on ? v[j][e] : 0.f);
    }
  }
  const float inv = 1.f / L;
  *reinterpret_cast<f32x4*>(a.out + (t * a.Hq + head) * D + 4 * part) = o * inv;
}

// Head sizes without a tiled kernel: one row (node, query head) by one wavefront, token after token,
// lanes over the dims.
template <typename E, int D>
__global__ __launch_bounds__(kWave) void tree_row_kernel(TreeArgs a) {
  constexpr int W = (D + kWave - 1) / kWave;
  const int lane = threadIdx.x, head = blockIdx.x, kvh = head / a.G;
  const int64_t t = blockIdx.y;
  const int seq = a.plan[lsh::plan_owners_at(a.S) + t];
  if (seq < 0 || seq >= a.S) return;
  const DraftSeq u = lsh::plan_seqs(a.plan)[seq];
  const uint64_t see = static_cast<uint64_t>(a.ancestors[t]);
  const int64_t* bt = a.bt + static_cast<int64_t>(seq) * a.max_blocks;
  const int64_t cap = static_cast<int64_t>(a.max_blocks) * a.bs, blocks = a.num_slots / a.bs;
  const int64_t len = u.ctx + u.nodes < cap ? u.ctx + u.nodes : cap;
  float q[W], acc[W], m = -1e30f, l = 0.f;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const int d = lane + kWave * w;
    float v = d < D ? a.q[(t * a.Hq + head) * D + d] : 0.f;
    if (a.q_mult && d < D) v = __fmul_rn(v, a.q_mult[head * D + d]);
    q[w] = v * (a.scale * kLog2e);
    acc[w] = 0.f;
  }
  for (int64_t p = 0; p < len; ++p) {
    if (p >= u.ctx && !(see >> (p - u.ctx) & 1)) continue;
    const int64_t id = bt[p / a.bs];
    if (id < 0 || id >= blocks) continue;
    const int64_t at = (id * a.bs + p % a.bs) * a.Hk + kvh;
    float s = 0.f, v[W], ks = 1.f, vs = 1.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const int d = lane + kWave * w;
      v[w] = 0.f;
      if (d < D) {
        s = __builtin_fmaf(q[w], static_cast<float>(static_cast<const E*>(a.kc)[at * D + d]), s);
        v[w] = static_cast<float>(static_cast<const E*>(a.vc)[at * D + d]);
      }
    }
    if constexpr (std::is_same_v<E, int8_t>) {
      ks = a.ks[at];
      vs = a.vs[at];
    }
    s = lsh::group_sum<kWave>(s) * ks;
    const float top = fmaxf(m, s), f = __builtin_amdgcn_exp2f(m - top), e = __builtin_amdgcn_exp2f(s - top);
    m = top;
    l = l * f + e;
#pragma unroll
    for (int w = 0; w < W; ++w) acc[w] = __builtin_fmaf(e * vs, v[w], acc[w] * f);
  }
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const int d = lane + kWave * w;
    if (d < D) a.out[(t * a.Hq + head) * D + d] = acc[w] / l;
  }
}

template <typename E, int D>
auto tiled_kernel(const TreeArgs& a) {
  if constexpr (std::is_same_v<E, float>) {
    // fp16 pieces where trees have more than 32 rows a kv head on average (208: 49 us against 83; 52: 106 against 120; 40: 114
    // against 127; 10: 169 against 136: with up to 32 rows three wavefronts only stage). Of trees that differ much the
    // average says less: one of 64 nodes among 31 single tokens takes 192 us, 137 in pieces; one single token among 7 trees 61
    // in pieces, 102 without.
    if constexpr (D == 128)
      if (a.T * a.G > kSplitRows * a.S) return tree_split_kernel<D>;
    return tree_f32_kernel<D>;
  } else {
    return tree_int8_kernel<D>;
  }
}

template <typename E>
void launch_tree(const TreeArgs& a, int64_t D, bool merge, hipStream_t st) {
  const dim3 items(static_cast<unsigned>(a.Hk), static_cast<unsigned>(std::min<int64_t>(a.items, lsh::plan_blocks(a.Hk))));
  const dim3 block(kWaves * kWave);
  if (D == 128 || D == 64) {
    if (D == 128)
      lsh::launch(tiled_kernel<E, 128>(a), items, block, 0, st, !merge, a);
    else
      lsh::launch(tiled_kernel<E, 64>(a), items, block, 0, st, !merge, a);
    if (!merge) return;
    const int64_t rows = kWaves * kWave / (D / 4);
    const dim3 grid(static_cast<unsigned>((a.T * a.Hq + rows - 1) / rows));
    if (D == 128)
      lsh::launch(tree_merge_kernel<128>, grid, block, 0, st, true, a);
    else
      lsh::launch(tree_merge_kernel<64>, grid, block, 0, st, true, a);
    return;
  }
  const dim3 grid(static_cast<unsigned>(a.Hq), static_cast<unsigned>(a.T));
  switch (D) {
    case 16: lsh::launch(tree_row_kernel<E, 16>, grid, dim3(kWave), 0, st, true, a); break;
    case 32: lsh::launch(tree_row_kernel<E, 32>, grid, dim3(kWave), 0, st, true, a); break;
    case 96: lsh::launch(tree_row_kernel<E, 96>, grid, dim3(kWave), 0, st, true, a); break;
    case 256: lsh::launch(tree_row_kernel<E, 256>, grid, dim3(kWave), 0, st, true, a); break;
    default: break;
  }
}

}  // namespace

extern "C" int64_t llmserve_paged_attention_tree_workspace_bytes(int64_t S, int64_t T, int64_t max_blocks,
                                                                 int64_t block_size, int64_t Hq, int64_t Hk,
                                                                 int64_t D) {
  if (Hq <= 0 || Hk <= 0 || Hq % Hk || (D != 64 && D != 128)) return 0;
  // one tile of no more than a block has one part (a second tile may begin anywhere in a block)
  if (S <= 1 && max_blocks * block_size <= lsh::kLeastBlock &&
      lsh::row_tiles(T < lsh::kMaxNodes ? T : lsh::kMaxNodes, Hq / Hk) <= 1)
    return 0;
  return llmserve_draft_plan_items(S, T, max_blocks, block_size, Hq / Hk, Hk) * Hk * lsh::kTreeRows * (D + 2) * 4;
}

extern "C" int llmserve_paged_attention_tree(const float* q, const void* k_cache, const void* v_cache,
                                             const float* k_scale, const float* v_scale, const int64_t* block_tables,
                                             const int64_t* ancestors, const void* plan, float* out, int64_t S,
                                             int64_t T, int64_t Hq, int64_t Hk, int64_t D, int64_t num_slots,
                                             int64_t max_blocks, int64_t block_size, float scale, const float* q_mult,
                                             void* workspace, int64_t workspace_bytes, void* stream) {
  LSH_CHECK(S >= 0 && T >= 0 && Hq >= 1 && Hk >= 1 && Hq % Hk == 0, "paged_attention_tree: bad shape");
  LSH_CHECK(D == 16 || D == 32 || D == 64 || D == 96 || D == 128 || D == 256,
            "paged_attention_tree: head_dim %lld not 16, 32, 64, 96, 128 or 256", (long long)D);
  if (S == 0 || T == 0) return LLMSERVE_OK;
  LSH_CHECK(block_size >= 1 && max_blocks >= 1 && num_slots >= block_size,
            "paged_attention_tree: empty block table or cache");
  LSH_CHECK(S < (1 << 16) && T < (1 << 16) && max_blocks < (1LL << 30) && block_size < (1LL << 30) &&
                max_blocks * block_size < (1LL << 30) && num_slots * Hk < (1LL << 31) && Hk <= 4096 && Hq / Hk <= 1024,
            "paged_attention_tree: batch, context or cache too large");
  LSH_CHECK(q && k_cache && v_cache && block_tables && ancestors && plan && out && (!k_scale == !v_scale),
            "paged_attention_tree: null pointer");
  LSH_CHECK(lsh::aligned16(q) && lsh::aligned16(k_cache) && lsh::aligned16(v_cache) && lsh::aligned16(out) &&
                lsh::aligned16(plan) && (q_mult == nullptr || lsh::aligned16(q_mult)),
            "paged_attention_tree: q, caches, plan, q_mult and out must be 16-byte aligned");
  LSH_CHECK(out + T * Hq * D <= q || q + T * Hq * D <= out,
            "paged_attention_tree: out must not overlap q (workgroups read rows that others have written)");
  const int64_t need = llmserve_paged_attention_tree_workspace_bytes(S, T, max_blocks, block_size, Hq, Hk, D);
  LSH_CHECK(need == 0 || (workspace != nullptr && workspace_bytes >= need && lsh::aligned16(workspace)),
            "paged_attention_tree: a 16-byte aligned workspace of %lld bytes is needed (%lld given)", (long long)need,
            (long long)workspace_bytes);
  const int64_t items = llmserve_draft_plan_items(S, T, max_blocks, block_size, Hq / Hk, Hk);
  LSH_CHECK(items < 65536 && (T * Hq + 1) * (D / 4) / 256 < (1LL << 31), "paged_attention_tree: batch too large");
  int bs_shift = -1;
  for (int sh = 0; sh < 30; ++sh)
    if ((1LL << sh) == block_size) bs_shift = sh;
  float* const part = static_cast<float*>(workspace);
  const TreeArgs a{q, k_cache, v_cache, k_scale, v_scale, block_tables, ancestors, static_cast<const int*>(plan),
                   q_mult, out, part, part + need / 4 / (D + 2) * D, num_slots, T, static_cast<int>(S),
                   static_cast<int>(Hq), static_cast<int>(Hk), static_cast<int>(Hq / Hk), static_cast<int>(max_blocks),
                   static_cast<int>(block_size), bs_shift, static_cast<int>(items), scale};
  hipStream_t st = lsh::as_stream(stream);
  if (k_scale != nullptr)
    launch_tree<int8_t>(a, D, need > 0, st);
  else
    launch_tree<float>(a, D, need > 0, st);
  return lsh::launch_status("paged_attention_tree");
}
