// Metadata of a step that verifies trees of drafted tokens, from lengths and parents on the device.
//
// Sequence s has ctx = context_lens[s] cached tokens and the nodes draft_start[s] ..
// draft_start[s + 1] of the flat [T] stream: node 0 its last token, the others drafts, parents[i]
// the parent of node i as an index into the tree (-1: a root). For node i:
//   ancestors = {i} + ancestors(parent)      as a 64-bit mask
//   position  = ctx + |ancestors| - 1        (its rotary position)
//   slot      = table[(ctx + i) / bs] * bs + (ctx + i) % bs   (where its K/V is written; -1: none)
// A parent that is not an earlier node of the tree makes the node a root. Rows of no tree (a tree's
// nodes past the 64th, rows before the first and behind the last sequence) get slot -1, the mask 0
// and position 0; the attention, verification and commit kernels leave them alone.
//
// One wavefront per sequence, a lane per node: the masks close in six doublings
// (mask |= mask[to], to = to[to]), all in registers. Every workgroup derives the work plan of the
// attention (draft.h) from all lengths by itself, so that no workgroup waits for another. Bound by its chain
// of dependent loads, sums and divisions: 7.7 us for one sequence, 9.6 for 128; the call takes 9.6, most of it on the host.
#include "draft.h"

namespace {

using lsh::DraftItem;
using lsh::DraftSeq;
using lsh::kWave;
constexpr int kWaves = 4, kThreads = kWaves * kWave;
constexpr int64_t kStartCost = 256;
constexpr int kSizes = 6, kSums = kSizes;

struct MetaArgs {
  const int64_t *ctx_lens, *start, *parents, *tables;
  int64_t T, max_blocks, bs;
  int S, G, Hk;
  int64_t blocks;    // most blocks of the plan
  int64_t capacity;  // most items
  int64_t *positions, *slots, *ancestors;
  int* plan;
};

__device__ __forceinline__ DraftSeq tree_of(const MetaArgs& a, int s) {
  auto clamp = [](int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : (v > hi ? hi : v); };
  DraftSeq d{};
  const int64_t first = clamp(a.start[s], 0, a.T);
  int64_t n = clamp(a.start[s + 1], first, a.T) - first;
  const int64_t cap = a.max_blocks * a.bs, c = clamp(a.ctx_lens[s], 0, cap);
  d.first = static_cast<int>(first);
  d.nodes = static_cast<int>(n > lsh::kMaxNodes ? lsh::kMaxNodes : n);
  d.ctx = static_cast<int>(c);
  d.tiles = static_cast<int>(lsh::row_tiles(d.nodes, a.G));
  d.len = static_cast<int>(c + d.nodes < cap ? c + d.nodes : cap);
  return d;
}

// Items of all tiles of a sequence whose first one begins d.off tokens into a block of Q.
__device__ __forceinline__ int64_t items_of(const DraftSeq& d, int64_t Q, int64_t cost) {
  int64_t n = 0, off = d.off;
  for (int r = 0; r < d.tiles; ++r) {
    n += lsh::cut_tile(off, d.len, Q, cost).items;
    off = (off + lsh::tile_span(d.len, Q, cost)) % Q;
  }
  return n;
}

// Sums over the workgroup, in place.
template <typename I, int N>
__device__ void block_sums(I (&v)[N], int64_t (*red)[kSums]) {
  static_assert(N <= kSums);
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) v[i] += __shfl_xor(v[i], d, kWave);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave][i] = v[i];
    v[i] = 0;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i)
    for (int w = 0; w < kWaves; ++w) v[i] += static_cast<I>(red[w][i]);
}

// Inclusive sums over the lanes.
__device__ __forceinline__ int64_t wave_scan(int64_t v) {
  const int lane = threadIdx.x % kWave;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int64_t o = __shfl_up(static_cast<long long>(v), d, kWave);
    v += lane >= d ? o : 0;
  }
  return v;
}

__global__ __launch_bounds__(kThreads) void draft_metadata_kernel(MetaArgs a) {
  __shared__ int64_t red[kWaves][kSums];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int s0 = static_cast<int>(blockIdx.x) * kWaves;

  // ---- the plan: as many blocks as the device has places, of as few whole units as make the line ------
  const int s = s0 + wave;
  const DraftSeq mine = static_cast<int>(threadIdx.x) < a.S ? tree_of(a, threadIdx.x) : DraftSeq{};
  auto each = [&](auto f) {  // this thread's sequences
    f(mine);
    for (int i = threadIdx.x + kThreads; i < a.S; i += kThreads) f(tree_of(a, i));
  };
  int64_t sums[3] = {};  // of all tiles: places in the line, tokens, tiles
  each([&](const DraftSeq& d) {
    sums[0] += d.tiles * lsh::whole_units(d.len);
    sums[1] += static_cast<int64_t>(d.tiles) * d.len;
    sums[2] += d.tiles;
  });
  block_sums(sums, red);
  // A start takes as long as some hundred tokens (8 to 15 us): counted, a workgroup with a part of two
  // sequences does not end after the others (attention of 208 fp32 rows 98 -> 83 us, 64 single int8 tokens 107 -> 104;
  // up to half of a share instead of a quarter: 16 trees of 26 nodes 55.7 -> 51.6). A share of no more than the least
  // block has no second part to speak of.
  const int64_t share = sums[0] / a.blocks, half = share / 2;
  int64_t cost = share <= lsh::kLeastBlock ? 0 : (half < kStartCost ? half : kStartCost);
  // Or whole blocks for every tile, of the smallest of a few sizes that leave enough of them, if they are no larger (7 trees of
  // 14 nodes over up to 78 tokens 34 -> 15 us, 30 of 10 over up to 858 37 -> 28, 16 of 26 54 -> 50).
  uint32_t size[kSizes];
#pragma unroll
  for (int k = 0; k < kSizes; ++k) {  // a tile's last block is half empty, or up to all of it
    const int64_t room = a.blocks - (3 + k) * sums[2] / 8;
    // (any size will do: no need for an exact quotient)
    const float q = room > 0 ? fminf(static_cast<float>(sums[1]) / static_cast<float>(room), 0x1p29f) : 0x1p29f;
    const int64_t units = lsh::whole_units(static_cast<int64_t>(q) + 1);
    size[k] = static_cast<uint32_t>(units > lsh::kLeastBlock ? units : lsh::kLeastBlock);
  }
  int64_t line_of[1] = {};     // the line with the starts
  uint32_t count[kSizes] = {};  // blocks at each size (2^13 of a tile and 2^22 of a thread stand for more)
  each([&](const DraftSeq& d) {
    line_of[0] += d.tiles * lsh::whole_units(d.len + cost);
#pragma unroll
    for (int k = 0; k < kSizes; ++k)
      count[k] = min(count[k] + d.tiles * min((static_cast<uint32_t>(d.len) + size[k] - 1) / size[k], 1u << 13), 1u << 22);
  });
  block_sums(count, red);
  if (cost > 0) block_sums(line_of, red);
  int64_t total = cost > 0 ? line_of[0] : sums[0];
  const int64_t even = lsh::whole_units((total + a.blocks - 1) / a.blocks);
  int64_t Q = even > lsh::kLeastBlock ? even : static_cast<int64_t>(lsh::kLeastBlock);
  bool whole = false;
#pragma unroll
  for (int k = 0; k < kSizes; ++k) {
    if (whole || size[k] > Q || count[k] > a.blocks) continue;
    whole = true;
    Q = size[k];
    cost = lsh::kWholeBlocks;
    total = count[k] * Q;
  }
  // Every wavefront goes through all sequences, 64 at a time, with running sums of the line and of the items,
  // and keeps what is its own.
  DraftSeq d{};
  int64_t line = 0, items = 0, block = 0;  // block: that the first tile begins in
  for (int i0 = 0; i0 < a.S; i0 += kWave) {
    DraftSeq e{};
    if (i0 + lane < a.S) e = tree_of(a, i0 + lane);
    const int64_t tokens = e.tiles * lsh::tile_span(e.len, Q, cost);
    const int64_t upto = wave_scan(tokens);
    e.off = static_cast<int>((line + upto - tokens) % Q);
    const int64_t n = items_of(e, Q, cost), upto_n = wave_scan(n);
    e.item0 = static_cast<int>(items + upto_n - n);
    if (s >= i0 && s < i0 + kWave) {
      d = s < a.S ? tree_of(a, s) : DraftSeq{};
      d.off = __shfl(e.off, s - i0, kWave);
      d.item0 = __shfl(e.item0, s - i0, kWave);
      block = __shfl(static_cast<long long>((line + upto - tokens) / Q), s - i0, kWave);
    }
    line += __shfl(static_cast<long long>(upto), kWave - 1, kWave);
    items += __shfl(static_cast<long long>(upto_n), kWave - 1, kWave);
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    a.plan[0] = static_cast<int>((total + Q - 1) / Q);
    a.plan[1] = static_cast<int>(items < a.capacity ? items : a.capacity);
    a.plan[2] = static_cast<int>(Q);
    a.plan[3] = static_cast<int>(cost);
  }
  if (s >= a.S) return;
  if (lane == 0) *const_cast<DraftSeq*>(lsh::plan_seqs(a.plan) + s) = d;
  DraftItem* const list = const_cast<DraftItem*>(lsh::plan_items(a.plan, a.S, a.T));
  int* const starts = a.plan + lsh::plan_starts_at(a.S, a.T, a.capacity);
  int64_t at = d.item0, off = d.off;
  for (int r = 0; r < d.tiles; ++r) {
    const lsh::TileCut cut = lsh::cut_tile(off, d.len, Q, cost);
    for (int64_t k = lane; k < cut.items; k += kWave) {
      const int64_t j = cut.first + k, lo = j * Q - off - (cost > 0 ? cost : 0), hi = lo + Q;
      if (at + k >= a.capacity || block + j >= a.blocks) break;
      list[at + k] = {s, r, static_cast<int>(lo > 0 ? lo : 0), static_cast<int>(hi < d.len ? hi : d.len),
                      d.first, d.nodes, d.ctx, static_cast<int>(cut.items)};
      if (j > 0 || off == 0) starts[block + j] = static_cast<int>(at + k);
    }
    at += cut.items;
    off += lsh::tile_span(d.len, Q, cost);
    block += off / Q;
    off %= Q;
  }

  int* owners = a.plan + lsh::plan_owners_at(a.S);
  // ---- the nodes ---------------------------------------------------------------------------------
  const int64_t t = static_cast<int64_t>(d.first) + lane;
  const bool on = lane < d.nodes;
  const int64_t p = on ? a.parents[t] : -1;
  int to = p >= 0 && p < lane ? static_cast<int>(p) : lane;
  uint64_t mask = 1ull << lane;
#pragma unroll
  for (int i = 0; i < 6; ++i) {
    mask |= static_cast<uint64_t>(__shfl(static_cast<long long>(mask), to, kWave));
    to = __shfl(to, to, kWave);
  }
  if (on) {
    const int64_t pos = static_cast<int64_t>(d.ctx) + lane, block = pos / a.bs;
    const int64_t id = block < a.max_blocks ? a.tables[s * a.max_blocks + block] : -1;
    a.positions[t] = d.ctx + __popcll(mask) - 1;
    a.slots[t] = id >= 0 ? id * a.bs + pos % a.bs : -1;
    a.ancestors[t] = static_cast<int64_t>(mask);
    owners[t] = s;
  }
  // rows of no tree: nodes past the 64th, rows before the first and behind the last sequence
  auto none = [&](int64_t from, int64_t to) {
    for (int64_t r = from + lane; r < to; r += kWave) {
      a.positions[r] = 0;
      a.slots[r] = -1;
      a.ancestors[r] = 0;
      owners[r] = -1;
    }
  };
  if (s == 0) none(0, d.first);
  none(d.first + d.nodes, s + 1 < a.S ? tree_of(a, s + 1).first : a.T);
}

// A batch without sequences: all of its rows belong to no tree.
__global__ __launch_bounds__(kThreads) void no_trees_kernel(int64_t T, int64_t* positions, int64_t* slots, int64_t* ancestors) {
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (t >= T) return;
  positions[t] = 0;
  slots[t] = -1;
  ancestors[t] = 0;
}

}  // namespace

extern "C" int64_t llmserve_draft_plan_items(int64_t S, int64_t T, int64_t max_blocks, int64_t block_size,
                                             int64_t G, int64_t Hk) {
  if (S <= 0 || T < 0 || max_blocks <= 0 || block_size <= 0 || G <= 0 || Hk <= 0) return 0;
  const int64_t nodes = T < S * lsh::kMaxNodes ? T : S * lsh::kMaxNodes;
  const int64_t tiles = nodes * G / lsh::kTreeRows + (S < nodes ? S : nodes);
  // every tile begins an item, and so does every block; and a tile has at most one item more than blocks of
  // the smallest size make it
  const int64_t most = (max_blocks * block_size + lsh::kLeastBlock - 1) / lsh::kLeastBlock + 1;
  const int64_t planned = lsh::plan_blocks(Hk) + tiles;
  return planned < tiles * most ? planned : tiles * most;
}

extern "C" int64_t llmserve_draft_plan_bytes(int64_t S, int64_t T, int64_t items, int64_t Hk) {
  return S < 0 || T < 0 || items < 0 || Hk < 0 ? 0 : 4 * lsh::plan_words(S, T, items, Hk);
}

extern "C" int llmserve_draft_metadata(const int64_t* context_lens, const int64_t* draft_start, const int64_t* parents,
                                       const int64_t* block_tables, int64_t S, int64_t T, int64_t max_blocks,
                                       int64_t block_size, int64_t G, int64_t Hk, int64_t* positions, int64_t* slots,
                                       int64_t* ancestors, void* plan, int64_t plan_bytes, void* stream) {
  LSH_CHECK(S >= 0 && T >= 0 && max_blocks >= 0 && block_size >= 1 && G >= 1 && Hk >= 1,
            "draft_metadata: bad sizes (S=%lld, T=%lld, max_blocks=%lld, block_size=%lld, G=%lld, Hk=%lld)",
            (long long)S, (long long)T, (long long)max_blocks, (long long)block_size, (long long)G, (long long)Hk);
  if (S == 0 && T == 0) return LLMSERVE_OK;
  if (S == 0) {
    LSH_CHECK(T < (1LL << 24), "draft_metadata: batch or context too large");
    LSH_CHECK(positions && slots && ancestors, "draft_metadata: null pointer");
    lsh::launch(no_trees_kernel, dim3(static_cast<unsigned>((T + kThreads - 1) / kThreads)), dim3(kThreads), 0, lsh::as_stream(stream),
                true, T, positions, slots, ancestors);
    return lsh::launch_status("draft_metadata");
  }
  LSH_CHECK(max_blocks >= 1, "draft_metadata: sequences without blocks");
  LSH_CHECK(S <= (1 << 16) && T < (1LL << 24) && max_blocks < (1LL << 30) && block_size < (1LL << 30) &&
                max_blocks * block_size < (1LL << 30) && G <= 1024 && Hk <= 4096,
            "draft_metadata: batch or context too large");
  LSH_CHECK(context_lens && draft_start && block_tables && plan && (T == 0 || (parents && positions && slots && ancestors)),
            "draft_metadata: null pointer");
  LSH_CHECK((T * G / lsh::kTreeRows + S) * (max_blocks * block_size + kStartCost) / lsh::plan_blocks(Hk) < (1LL << 30),
            "draft_metadata: batch times context too large");
  const int64_t items = llmserve_draft_plan_items(S, T, max_blocks, block_size, G, Hk);
  LSH_CHECK(lsh::aligned16(plan) && plan_bytes >= 4 * lsh::plan_words(S, T, items, Hk),
            "draft_metadata: a 16-byte aligned plan of %lld bytes is needed (%lld given)",
            (long long)(4 * lsh::plan_words(S, T, items, Hk)), (long long)plan_bytes);
  const MetaArgs a{context_lens, draft_start, parents, block_tables, T, max_blocks, block_size, static_cast<int>(S),
                   static_cast<int>(G), static_cast<int>(Hk), lsh::plan_blocks(Hk), items, positions, slots, ancestors,
                   static_cast<int*>(plan)};
  lsh::launch(draft_metadata_kernel, dim3(static_cast<unsigned>((S + kWaves - 1) / kWaves)), dim3(kThreads), 0,
              lsh::as_stream(stream), true, a);
  return lsh::launch_status("draft_metadata");
}
