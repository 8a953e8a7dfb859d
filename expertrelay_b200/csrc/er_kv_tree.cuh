// er_kv_tree.cuh -- what the kernels of er_kv_tree share: the trees of a call
// as the device finds them.
//
// Tree t's nodes are rows starts[t] .. starts[t + 1] - 1 of the queries, their
// keys and values the places lens[t] + i of sequence seqs[t]. Node i sees the
// first lens[t] places, its ancestors (parents[], within the tree) and itself.
#pragma once

#include "er_kv.cuh"

namespace er {

constexpr int kMaxTrees = 4096, kMaxNodes = 256;

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

}  // namespace er
