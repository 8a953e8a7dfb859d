// er_kv_tree.cuh -- what the kernels of er_kv_tree share: the trees of a call
// as the device finds them.
//
// Tree t's nodes are rows starts[t] .. starts[t + 1] - 1 of the queries, their
// keys and values the places lens[t] + i of sequence seqs[t]. Node i sees the
// first lens[t] places, its ancestors (parents[], within the tree) and itself.
#pragma once

#include <cuda.h>

#include "er_kv_attend.cuh"

namespace er {

constexpr int kMaxTrees = 4096, kMaxNodes = 256;
constexpr int kTreeRows = 128;  // of a matrix product
constexpr int kTreeChannels = 128;  // of the values, at most, that a unit has

// A unit whose tiles several CTAs share: the first of them writes it, the join reads it.
struct TreeCut {
  int first, head, q0, live;  // live 0: none begins here and ends behind
  int tiles, ch0;
  long long begin, total;  // the unit's place in the line, and the line's length
};

struct TreeArgs {
  KvView kv;
  const void* q;
  long long q_stride;
  void* out;
  int rows, heads, group;  // group: queries per key head
  int trees;
  const int32_t *starts, *parents, *seqs, *lens;
  float scale;             // scale * log2(e)
  int* status;
  int q_wide;              // rows of q on 16-byte boundaries
  int q_flip, q_zero;      // the scale was negative, or zero: queries change their sign, or are zero
  int tile;                // keys of a tile
  int block_rows;          // query rows of a unit at most
  int channels, halves;    // of the values: those of a unit, units beside each other for all of them
  int box_rows;            // positions that a copy takes: they lie in one page wherever it begins
  int grid;                // CTAs of the attention kernel
  int piece_rows;          // rows that a piece has room for
  TreeCut* cut;            // [grid]
  float* part_ml;          // [2 grid][piece_rows][2]: m, l of a CTA's first piece and of one that begins in it
  float* part_o;           // [2 grid][piece_rows][channels]
};

// A tree: its rows first .. first + nodes - 1 and its context. Where its rows
// are not known there are none (nodes 0); where something else is wrong with
// it they are spoilt (bad).
struct Tree {
  int first, nodes, len, seq;
  int bad;  // ER_KV_BAD_* bits
};

__device__ __forceinline__ Tree kv_tree(const TreeArgs& a, int t) {
  Tree e;
  e.first = a.starts[t];  // loads that wait for none of each other
  const int end = a.starts[t + 1];
  e.len = a.lens[t];
  e.seq = a.seqs ? a.seqs[t] : t;
  e.nodes = end - e.first;
  e.bad = 0;
  if (e.first < 0 || end < e.first || end > a.rows) {
    e.first = e.nodes = 0;
    e.bad = ER_KV_BAD_TREE;
  } else if (e.nodes > kMaxNodes) {
    e.bad = ER_KV_BAD_TREE;
  } else if (e.seq < 0 || e.seq >= a.kv.seqs) {
    e.bad = ER_KV_BAD_SEQ;
  } else if (e.len < 0 || (long long)e.len + e.nodes > min(a.kv.capacity(), 0x7fff0000ll)) {
    e.bad = ER_KV_BAD_LENGTH;
  }
  return e;
}


// The line that the CTAs share. A unit is a block of at most block_rows query
// rows (nodes x group, in equal blocks) of one key head of a tree, and of at
// most 128 channels of its values; it takes its tiles and kTreeCost of the
// line, for its queries, masks and result.
constexpr int kTreeCost = 4, kTreeMinShare = 2;

struct TreeUnits {
  int rows, blocks, per, units, tiles;  // query rows of a key head, blocks of them, rows of a block
};
__device__ __forceinline__ TreeUnits tree_units(const TreeArgs& a, const Tree& e) {
  TreeUnits u = {};
  if (e.bad || e.nodes == 0) return u;
  u.rows = e.nodes * a.group;
  u.blocks = (u.rows + a.block_rows - 1) / a.block_rows;
  u.per = (u.rows + u.blocks - 1) / u.blocks;
  u.units = u.blocks * a.halves * a.kv.kv_heads;
  u.tiles = (e.len + e.nodes + a.tile - 1) / a.tile;
  return u;
}

__device__ __forceinline__ int tree_shares(const TreeArgs& a, long long total) {
  return total < (long long)a.grid * kTreeMinShare ? ((int)total + kTreeMinShare - 1) / kTreeMinShare : a.grid;
}

// A CTA's run: the places from..to of the line, and the tree that `from` lies in with its place.
struct TreeRun {
  long long from, to, total, at;
  int t;
};
struct TreeScratch {
  long long cost[32];
};

// All threads; every CTA sums the trees' costs itself. Ends with a barrier.
__device__ __forceinline__ void tree_run(const TreeArgs& a, TreeRun& run, TreeScratch& s) {
  const int threads = blockDim.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per = (a.trees + threads - 1) / threads;
  const int t0 = min(a.trees, (int)threadIdx.x * per), t1 = min(a.trees, t0 + per);
  long long mine = 0;
  for (int t = t0; t < t1; ++t) {
    const Tree e = kv_tree(a, t);
    if (blockIdx.x == 0 && e.bad) kv_report(a.status, e.bad);
    const TreeUnits u = tree_units(a, e);
    mine += (long long)u.units * (u.tiles + kTreeCost);
  }
  long long in = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long up = __shfl_up_sync(0xffffffffu, in, o);
    if (lane >= o) in += up;
  }
  if (lane == 31) s.cost[warp] = in;
  if (threadIdx.x == 0) run = TreeRun{};
  __syncthreads();
  long long total = 0;
  for (int w = 0; w < threads / 32; ++w) {
    if (w == warp) in += total;
    total += s.cost[w];
  }
  if (total > 0) {
    const int shares = tree_shares(a, total);
    if ((int)blockIdx.x < shares) {
      const long long from = kv_share_start(total, shares, blockIdx.x), to = kv_share_start(total, shares, blockIdx.x + 1);
      long long at = in - mine;
      if (from >= at && from < in) {
        int t = t0;
        for (; t < t1; ++t) {
          const TreeUnits u = tree_units(a, kv_tree(a, t));
          const long long c = (long long)u.units * (u.tiles + kTreeCost);
          if (from < at + c) break;
          at += c;
        }
        run = TreeRun{from, to, total, at, t};
      }
    }
  }
  __syncthreads();
}

// The units of a run that have tiles in it, one after another: tiles lo .. hi - 1 of `tiles`.
struct TreeWalk {
  const TreeArgs& a;
  const TreeRun& run;
  int t, unit;
  Tree e;
  TreeUnits u;
  long long pos;  // where the unit begins in the line
  int lo, hi, tiles, head, q0, live, ch0;
  int most;  // replicas

  __device__ __forceinline__ TreeWalk(const TreeArgs& args, const TreeRun& r, int most_replicas)
      : a(args), run(r), most(most_replicas) {}

  __device__ __forceinline__ bool look() {  // from unit `unit` of tree t at pos on: the next one with tiles in the run
    for (;;) {
      if (pos >= run.to) return false;
      if (unit >= u.units) {
        do {
          if (++t >= a.trees) return false;
          e = kv_tree(a, t);
          u = tree_units(a, e);
        } while (u.units == 0);
        unit = 0;
      }
      const long long first = pos + kTreeCost;
      lo = run.from > first ? (int)(run.from - first < u.tiles ? run.from - first : u.tiles) : 0;
      hi = run.to < first + u.tiles ? (int)(run.to > first ? run.to - first : 0) : u.tiles;
      if (hi > lo) break;
      pos += u.tiles + kTreeCost;
      ++unit;
    }
    tiles = u.tiles;
    const int beside = u.blocks * a.halves, rest = unit % beside;
    head = unit / beside;
    q0 = rest / a.halves * u.per;
    ch0 = rest % a.halves * kTreeChannels;
    live = min(u.per, u.rows - q0);
    return true;
  }
  __device__ __forceinline__ bool begin() {
    if (run.total == 0 || run.from == run.to) return false;
    t = run.t;
    e = kv_tree(a, t);
    u = tree_units(a, e);
    const int c = u.tiles + kTreeCost;
    unit = (int)kv_div(run.from - run.at, c);
    pos = run.at + (long long)unit * c;
    return look();
  }
  __device__ __forceinline__ bool next() {
    pos += u.tiles + kTreeCost;
    ++unit;
    return look();
  }
  // Few rows are taken several times, each for its share of a tile's keys, so that all of the lanes of the
  // scores' memory have work.
  __device__ __forceinline__ int replicas() const {
    return most >= 4 && live <= 32 ? 4 : most >= 2 && live <= 16 * most ? 2 : 1;
  }
};

// What a launch of the attention kernel takes: keys of a tile, query rows of a
// unit, its channels and how many units have the others.
struct TreeLaunch {
  int tile, rows, channels, halves;
};
// er_kv_tree_bf16.cu and er_kv_tree_f32.cu: for caches of either type
TreeLaunch tree_shape_bf16(int d, int q_dtype);
TreeLaunch tree_shape_f32(int d);
template <typename S>
constexpr TreeLaunch tree_shape() {
  return TreeLaunch{S::TK, S::ROWS, S::VD, S::DP / S::VD};
}
int tree_bf16(const TreeArgs& a, int q_dtype, const CUtensorMap* maps, cudaStream_t st);
int tree_f32(const TreeArgs& a, int q_dtype, cudaStream_t st);

}  // namespace er
