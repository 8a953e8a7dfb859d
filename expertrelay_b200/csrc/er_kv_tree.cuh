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
constexpr int kTreeChannels = 128;  // of the values, at most, that a unit has

// A unit whose tiles several CTAs share: the first of them writes it, the join reads it.
struct TreeCut {
  int first, head, q0, live;  // live 0: none begins here and ends behind; -1: a wait of the CTA gave up
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
  int tile_shift;          // log2 of a tile's keys
  int unit_cost;           // what a unit takes beside its tiles, in tiles
  int block_rows, block_shift;  // query rows of a unit at most (a power of two), and its log2
  int channels, halves;    // of the values: those of a unit, units beside each other for all of them
  int box_rows;            // positions that a copy takes: they lie in one page wherever it begins
  int grid;                // CTAs of the attention kernel
  int piece_rows;          // rows that a piece has room for
  TreeCut* cut;            // [grid]
  float* part_ml;          // [2 grid][piece_rows][2]: m, l of a CTA's first piece and of one that begins in it
  float* part_o;           // [2 grid][piece_rows][channels]
  unsigned long long wait_ns;  // limit of a wait
  int stall;               // test hook (er_kv_tree_test_stall): a wait at a CTA's end that runs out
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
// most 128 channels of its values; it takes its tiles and unit_cost of the
// line, for its queries, masks and result.
constexpr int kTreeMinShare = 2;

// the node that a key head's query row belongs to
__device__ __forceinline__ int tree_node(const TreeArgs& a, int q) { return a.group == 1 ? q : q / a.group; }

struct TreeUnits {
  int rows, blocks, per, units, tiles;  // query rows of a key head, blocks of them, rows of a block
};
__device__ __forceinline__ TreeUnits tree_units(const TreeArgs& a, const Tree& e) {
  TreeUnits u = {};
  if (e.bad || e.nodes == 0) return u;
  u.rows = e.nodes * a.group;  // divisions are left out where they can be: every warp comes here at its start
  u.blocks = (u.rows + a.block_rows - 1) >> a.block_shift;
  u.per = u.blocks == 1 ? u.rows : (u.rows + u.blocks - 1) / u.blocks;
  u.units = u.blocks * a.halves * a.kv.kv_heads;
  u.tiles = (e.len + e.nodes + (1 << a.tile_shift) - 1) >> a.tile_shift;
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
    mine += (long long)u.units * (u.tiles + a.unit_cost);
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
          const long long c = (long long)u.units * (u.tiles + a.unit_cost);
          if (from < at + c) break;
          at += c;
        }
        run = TreeRun{from, to, total, at, t};
      }
    }
  }
  __syncthreads();
}

// The units of a run that have tiles in it, one after another. Every warp goes
// its own way through them, in shared memory and by one copy of the code: each
// copy would be fetched for the first time in every launch.
struct TreeWalk {
  int t, unit;
  Tree e;
  TreeUnits u;
  long long pos;    // where the unit begins in the line
  int lo, hi;       // its tiles in the run, of u.tiles
  int head, q0, live, ch0;
  int replicas;
};

// The warp's next unit (its first one where `first`); false where there is none. `most`: replicas.
static __device__ __noinline__ bool tree_next(const TreeArgs& a, const TreeRun& run, TreeWalk* walk, bool first, int most) {
  if (run.total == 0 || run.from == run.to) return false;
  TreeWalk w;
  if (first) {
    w.t = run.t;
    w.e = kv_tree(a, w.t);
    w.u = tree_units(a, w.e);
    const int c = w.u.tiles + a.unit_cost;
    w.unit = (int)kv_div(run.from - run.at, c);
    w.pos = run.at + (long long)w.unit * c;
  } else {
    w = *walk;
    w.pos += w.u.tiles + a.unit_cost;
    ++w.unit;
  }
  for (;;) {
    if (w.pos >= run.to) return false;
    if (w.unit >= w.u.units) {
      do {
        if (++w.t >= a.trees) return false;
        w.e = kv_tree(a, w.t);
        w.u = tree_units(a, w.e);
      } while (w.u.units == 0);
      w.unit = 0;
    }
    const long long tile0 = w.pos + a.unit_cost;
    w.lo = run.from > tile0 ? (int)(run.from - tile0 < w.u.tiles ? run.from - tile0 : w.u.tiles) : 0;
    w.hi = run.to < tile0 + w.u.tiles ? (int)(run.to > tile0 ? run.to - tile0 : 0) : w.u.tiles;
    if (w.hi > w.lo) break;
    w.pos += w.u.tiles + a.unit_cost;
    ++w.unit;
  }
  const int beside = w.u.blocks * a.halves;
  w.head = beside == 1 ? w.unit : w.unit / beside;
  const int rest = w.unit - w.head * beside;
  w.q0 = (a.halves == 2 ? rest >> 1 : rest) * w.u.per;
  w.ch0 = a.halves == 2 ? (rest & 1) * kTreeChannels : 0;
  w.live = min(w.u.per, w.u.rows - w.q0);
  // Few rows are taken several times, each for its share of a tile's keys, so that all of the lanes of the
  // scores' memory have work.
  w.replicas = most >= 4 && w.live <= 32 ? 4 : most >= 2 && w.live <= 16 * most ? 2 : 1;
  __syncwarp();
  if ((threadIdx.x & 31) == 0) *walk = w;
  __syncwarp();
  return true;
}

// What a launch of the attention kernel takes: keys of a tile, query rows of a
// unit, its channels and how many units have the others.
struct TreeLaunch {
  int tile, rows, channels, halves;
  int box_rows, box_channels;  // of a copy, at most (0: none are issued)
};
// er_kv_tree_bf16.cu and er_kv_tree_f32.cu: for caches of either type
TreeLaunch tree_shape_bf16(int d, int q_dtype);
TreeLaunch tree_shape_f32(int d);
template <typename S>
constexpr TreeLaunch tree_shape() {
  return TreeLaunch{S::TK, S::ROWS, S::VD, S::DP / S::VD, S::KP == 1 ? S::TK : S::kRaw ? S::kRawRows : 0,
                    S::KP == 1 ? 64 : S::DP};
}
int tree_bf16(const TreeArgs& a, int q_dtype, const CUtensorMap* maps, cudaStream_t st);
int tree_f32(const TreeArgs& a, int q_dtype, const CUtensorMap* maps, cudaStream_t st);

}  // namespace er
