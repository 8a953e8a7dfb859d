// er_kv_attend.cuh -- what the kernels of er_kv_attend share: the division of
// the work, the walk over a row's pages, and the joining of partial results.
//
// out = sum_j p_j v_j / sum_j p_j, p_j = 2^(s_j - m), s_j = scale log2(e) q.k_j,
// is one pass over the keys with a running maximum m: a piece of the keys
// leaves (m, l = sum p, o = sum p v), and pieces join by
//   m = max m_i, l = sum l_i 2^(m_i - m), o = sum o_i 2^(m_i - m).
// Each key and value byte is used for 2 G flop (G queries a key head), so
// memory bounds it, and every SM has to stream an equal share however the
// lengths fall: the keys of all (row, key head) units lie in one line of
// tiles, and each CTA takes an equal run of it. The lengths are read on the
// device, so a captured graph serves any lengths that its tables hold.
#pragma once

#include "er_kv.cuh"

namespace er {

constexpr int kKvMaxLen = 0x7fff0000;  // positions stay ints with a tile's keys added
constexpr int kKvSegment = 8;           // keys that are looked up together where pages allow

// A unit whose tiles several CTAs share: the first of them writes it, the join reads it.
struct CutUnit {
  int row, head, g0;  // row -1: none begins here and ends behind
  int tiles;
  long long begin, total;  // the unit's place in the line, and the line's length
};

struct AttendArgs {
  KvView kv;
  const void* q;
  long long q_stride;
  void* out;
  int rows, heads, group;      // group: queries per key head
  int blocks;                  // head blocks a group is taken in
  const int32_t* seqs;
  const int32_t* lens;
  float scale;                 // scale * log2(e)
  const int32_t* pages;        // optional page lists [rows, kv_heads, max_pages]
  const int32_t* counts;
  int max_pages;
  int tile;                    // keys a tile: warps a CTA * keys of a warp's chunk
  int min_share;               // the least share of the line worth a CTA
  int* status;
  // scan entries: rows, or (row, key head) pairs when each has its own page list
  int entries, units;          // units of one entry: the tiles repeat that often
  CutUnit* cut;                // [grid] the unit that begins in a CTA's run and ends behind it
  float* part_ml;              // [2 grid][GB][2]: m, l of a CTA's first and last piece
  float* part_o;               // [2 grid][GB][d]
  int grid;                    // CTAs of the attention kernel
  int cluster;                 // a cluster per unit instead of shares of the line
  float* scores;               // optional [rows][kv_heads][mass_len][group], log2 units
  float* lse;                  // with scores: [rows][heads], log2 units
  float* mass;
  long long mass_row_stride, mass_head_stride;
  int mass_len;
};

// What an entry has: its keys (0 when something is wrong with it).
struct Entry {
  int n, len, seq;
  int bad;  // ER_KV_BAD_* bits
};

__device__ __forceinline__ Entry kv_entry(const AttendArgs& a, int x) {
  const int row = a.pages ? x / a.kv.kv_heads : x;
  Entry e;
  e.seq = a.seqs ? a.seqs[row] : row;  // three loads, none waiting for another
  e.len = a.lens[row];
  const int c = a.pages ? a.counts[x] : 0;
  e.n = a.pages ? (int)((uint32_t)c * a.kv.page_size) : e.len;  // of a page list, positions behind len are left out key by key
  e.bad = 0;
  if (e.seq < 0 || e.seq >= a.kv.seqs)
    e.bad = ER_KV_BAD_SEQ;
  else if (e.len < 0 || e.len > kKvMaxLen || e.len > a.kv.capacity() || (a.scores && e.len > a.mass_len))
    e.bad = ER_KV_BAD_LENGTH;
  else if (a.pages && (c < 0 || c > a.max_pages || (long long)c * a.kv.page_size > kKvMaxLen))
    e.bad = ER_KV_BAD_LENGTH;
  if (e.bad) e.n = 0;
  return e;
}

__device__ __forceinline__ int kv_tiles(const AttendArgs& a, int n) { return (n + a.tile - 1) / a.tile; }

// The line that the CTAs share: a unit of c > 0 tiles takes kUnitCost + c of
// it, for its queries, the joining of its warps and its result cost about
// that many tiles beside the tiles themselves. (48 rows of 1 .. 4097 keys and
// 16 heads, shares by tiles alone: the CTAs with the short rows ran on for 21 % of
// the kernel after the others.)
constexpr int kUnitCost = 3;
__device__ __forceinline__ int kv_cost(int tiles) { return tiles ? tiles + kUnitCost : 0; }

// 64-bit division as a call (inlined, each is a hundred instructions that a
// short launch would fetch for the first time), 32-bit where that is enough.
static __device__ __noinline__ long long kv_div(long long a, long long b) {
  if (((a | b) >> 32) == 0) return (uint32_t)a / (uint32_t)b;
  return a / b;
}
__device__ __forceinline__ int kv_shares(const AttendArgs& a, long long total) {
  return total < (long long)a.grid * a.min_share ? ((int)total + a.min_share - 1) / a.min_share : a.grid;
}
// where share i begins, and the share that place x lies in
__device__ __forceinline__ long long kv_share_start(long long total, int shares, int i) {
  return kv_div(total * i, shares);
}
__device__ __forceinline__ int kv_share_of(long long total, int shares, long long x) {
  return (int)kv_div((x + 1) * shares - 1, total);
}

// A CTA's run of tiles: the first one (entry x, unit u of it, tile t of the
// `tiles` of that unit), how many, and where the first one's unit begins in
// the line of length `total`.
struct Run {
  int x, u, t, tiles;
  Entry e;
  long long left, begin, total;
};
struct RunScratch {  // shared memory of kv_run
  long long cost[8], tiles[8];  // by warp
  Run run;
  long long before[2];  // tiles before the run, and before its end
};

// Every CTA sums the entries' costs itself (a few loads a thread) and finds
// its share's two ends.
__device__ __forceinline__ Run kv_run(const AttendArgs& a, RunScratch& s) {
  const int threads = blockDim.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    a.cut[blockIdx.x].row = -1;
    s.before[0] = s.before[1] = 0;
  }
  if (a.entries == 1) {  // nothing to sum
    Run r = {};
    r.e = kv_entry(a, 0);
    if (blockIdx.x == 0 && threadIdx.x == 0 && r.e.bad) kv_report(a.status, r.e.bad);
    r.tiles = kv_tiles(a, r.e.n);
    const int k = kv_cost(r.tiles);
    r.total = (long long)k * a.units;
    if (k == 0) return r;
    const int shares = kv_shares(a, r.total);
    if ((int)blockIdx.x >= shares) return r;
    const long long at = kv_share_start(r.total, shares, blockIdx.x), to = kv_share_start(r.total, shares, blockIdx.x + 1);
    r.u = (int)kv_div(at, k);
    r.begin = (long long)r.u * k;
    r.t = max(0, (int)(at - r.begin) - kUnitCost);
    const int v = (int)kv_div(to, k);
    r.left = (long long)v * r.tiles + max(0, (int)(to - (long long)v * k) - kUnitCost) - ((long long)r.u * r.tiles + r.t);
    return r;
  }
  const int per = (a.entries + threads - 1) / threads;
  const int x0 = min(a.entries, (int)threadIdx.x * per), x1 = min(a.entries, x0 + per);
  long long cost = 0, tiles = 0;
  Entry e = {};
#pragma unroll 2
  for (int x = x0; x < x1; ++x) {
    e = kv_entry(a, x);
    const int c = kv_tiles(a, e.n);
    tiles += c;
    cost += kv_cost(c);
    if (blockIdx.x == 0 && e.bad) kv_report(a.status, e.bad);
  }
  const long long my_cost = cost, my_tiles = tiles;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long uc = __shfl_up_sync(0xffffffffu, cost, o), ut = __shfl_up_sync(0xffffffffu, tiles, o);
    if (lane >= o) {
      cost += uc;
      tiles += ut;
    }
  }
  if (lane == 31) {
    s.cost[warp] = cost;
    s.tiles[warp] = tiles;
  }
  __syncthreads();
  long long all = 0, all_tiles = 0;
#pragma unroll 1
  for (int w = 0; w < threads / 32; ++w) {
    if (w == warp) {
      cost += all;
      tiles += all_tiles;
    }
    all += s.cost[w];
    all_tiles += s.tiles[w];
  }
  Run r = {};
  r.total = all * a.units;
  if (r.total == 0) return r;
  const int shares = kv_shares(a, r.total);
  if ((int)blockIdx.x >= shares) return r;
  // this thread's entries hold the line from ex to in; `tb` tiles lie before them
  const long long ex = (cost - my_cost) * a.units, in = cost * a.units, tb = (tiles - my_tiles) * a.units;
#pragma unroll 1
  for (int end = 0; end < 2; ++end) {
    const long long at = kv_share_start(r.total, shares, blockIdx.x + end);
    if (at == r.total && threadIdx.x == 0) s.before[1] = all_tiles * a.units;
    if (at < ex || at >= in) continue;
    long long rest = at - ex, before = tb;
#pragma unroll 1
    for (int x = x0; x < x1; ++x) {
      if (per > 1) e = kv_entry(a, x);
      const int c = kv_tiles(a, e.n), k = kv_cost(c);
      if (rest < (long long)k * a.units) {
        const int u = (int)kv_div(rest, k), in_unit = (int)(rest - (long long)u * k), t = max(0, in_unit - kUnitCost);
        s.before[end] = before + (long long)u * c + t;
        if (end == 0) s.run = Run{x, u, t, c, e, 0, at - in_unit, r.total};
        break;
      }
      rest -= (long long)k * a.units;
      before += (long long)c * a.units;
    }
  }
  __syncthreads();
  r = s.run;
  r.left = s.before[1] - s.before[0];
  return r;
}

// 2^(m_i - m) of a piece, 0 for a piece without keys or of -inf scores alone.
__device__ __forceinline__ float piece_weight(float mi, float m) { return mi == -INFINITY ? 0.f : exp2f(mi - m); }

// With few units, each is a cluster's: its CTAs take an eighth of the tiles
// each and join their pieces through one another's shared memory, so there is
// no line to divide, no workspace and no second launch.
__device__ __forceinline__ float4 cluster_load4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

__device__ __forceinline__ Run kv_cluster_run(const AttendArgs& a) {
  Run r = {};
  const int unit = blockIdx.x / kClusterCtas, rank = cluster_rank();
  r.x = unit / a.units;
  r.u = unit % a.units;
  r.e = kv_entry(a, r.x);
  if (r.e.bad && r.u == 0 && rank == 0 && threadIdx.x == 0) kv_report(a.status, r.e.bad);
  r.tiles = kv_tiles(a, r.e.n);
  r.t = (int)((long long)r.tiles * rank / kClusterCtas);
  r.left = (int)((long long)r.tiles * (rank + 1) / kClusterCtas) - r.t;
  return r;
}

// Four results of query g of a unit, from their weighted sum and the weights' sum.
template <typename TQ>
__device__ __forceinline__ void kv_store4(TQ* to, float4 acc, float sum) {
  const float inv = 1.f / sum;
  const bool none = sum == 0.f;  // no key, or scores of -inf alone
  float v[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = none ? 0.f : v[e];
  if constexpr (sizeof(TQ) == 4) {
    *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    __nv_bfloat162 lo = __floats2bfloat162_rn(v[0], v[1]), hi = __floats2bfloat162_rn(v[2], v[3]);
    uint2 raw = make_uint2(*reinterpret_cast<uint32_t*>(&lo), *reinterpret_cast<uint32_t*>(&hi));
    *reinterpret_cast<uint2*>(to) = raw;
  }
}
__device__ __forceinline__ void fma4(float4& acc, float4 x, float by) {
  acc.x = fmaf(x.x, by, acc.x);
  acc.y = fmaf(x.y, by, acc.y);
  acc.z = fmaf(x.z, by, acc.z);
  acc.w = fmaf(x.w, by, acc.w);
}

// The cluster's pieces joined: in every CTA's shared memory, `ml` [heads][2]
// and `o` [heads][pitch]. Each CTA writes an eighth of the unit's results.
template <typename TQ>
__device__ __forceinline__ void kv_cluster_join(const AttendArgs& a, const Run& r, int gb, const float* ml,
                                                const float* o, int pitch) {
  cluster_sync();
  const int head = a.pages ? r.x % a.kv.kv_heads : r.u / a.blocks, row = a.pages ? r.x / a.kv.kv_heads : r.x;
  const int d = a.kv.d, g0 = r.u % a.blocks * gb, live_g = min(gb, a.group - g0), cols = d / 4;
  const uint32_t ml0 = smem_addr(ml), o0 = smem_addr(o);
#pragma unroll 1
  for (int i = threadIdx.x * kClusterCtas + cluster_rank(); i < live_g * cols; i += blockDim.x * kClusterCtas) {
    const int g = i / cols, col = i - g * cols;
    float2 p[kClusterCtas];
    float4 x[kClusterCtas];
#pragma unroll
    for (int k = 0; k < kClusterCtas; ++k) {
      p[k] = cluster_load2(cluster_addr(ml0 + g * 8, k));
      x[k] = cluster_load4(cluster_addr(o0 + (g * pitch + col * 4) * 4, k));
    }
    float top = -INFINITY, sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < kClusterCtas; ++k) top = fmaxf(top, p[k].x);
#pragma unroll
    for (int k = 0; k < kClusterCtas; ++k) {
      const float by = piece_weight(p[k].x, top);
      sum = fmaf(p[k].y, by, sum);  // a spoiled piece's sum is NaN
      fma4(acc, x[k], by);
    }
    if (r.e.bad) sum = __int_as_float(0x7fc00000);
    const long long at = (long long)row * a.heads + head * a.group + g0 + g;
    kv_store4((TQ*)a.out + at * d + col * 4, acc, sum);
    if (a.scores && col == 0) a.lse[at] = sum == 0.f ? INFINITY : top + log2f(sum);
  }
  cluster_sync();  // no CTA's shared memory goes before all have read it
}

// What the arithmetic of a tile needs to know, left by the warp when it
// issues the tile's copies.
struct __align__(16) StageInfo {
  uint32_t keys;  // the chunk's keys that exist
  int bad;        // whether one has a bad page
  int t, tiles;   // the tile, and its unit's tiles
  int row, head, g0;
  int pad;
};

// A warp's walk over its run, a chunk of KEYS keys each tile, ahead of the
// arithmetic. WHOLE: page_size is a multiple of 8, so each 8 keys lie in one
// page: the lanes hold the pages of the next tiles' eights. Otherwise lane i
// holds the page of the next chunk's key i, loaded a tile ahead of its use.
template <bool WHOLE, int KEYS>
struct Walk {
  static constexpr int kSegs = KEYS / kKvSegment, kWindow = 32 / kSegs;  // eights of a chunk, tiles that are held
  int x, u, t, tiles, head, lane, warp;
  Entry e;
  long long ahead;  // tiles not yet taken
  int win;          // WHOLE: the first tile that is held
  int page;         // -1: no key, -2: a bad page
  int slot;         // of the (first) key in its page
  int live;         // WHOLE: keys of the eight

  __device__ __forceinline__ Walk(const AttendArgs& a, const Run& r)
      : x(r.x), u(r.u), t(r.t), tiles(r.tiles), lane(threadIdx.x & 31), warp(threadIdx.x >> 5), e(r.e), ahead(r.left) {
    head = a.pages ? x % a.kv.kv_heads : u / a.blocks;
    look(a);
  }

  // loads the pages of the tiles' eights (of the chunk's keys) from tile t on
  __device__ __forceinline__ void look(const AttendArgs& a) {
    win = t;
    page = -1;
    slot = live = 0;
    const int j = warp * KEYS + (WHOLE ? (t + lane / kSegs) * a.tile + lane % kSegs * kKvSegment : t * a.tile + lane);
    if (j >= e.n || j < 0 || (!WHOLE && lane >= KEYS)) return;
    int o = a.kv.ordinal(j);
    slot = j - o * a.kv.page_size;
    live = min(e.n - j, kKvSegment);
    if (a.pages) {
      o = a.pages[(long long)x * a.max_pages + o];
      if (o < 0 || o >= a.kv.width) {
        page = -2;
        return;
      }
      const long long left = e.len - ((long long)o * a.kv.page_size + slot);
      live = left < live ? (int)left : live;
      if (live <= 0) {
        live = 0;
        return;
      }
    }
    page = a.kv.pages_of(e.seq)[o];
    if (page < 0 || page >= a.kv.num_pages) page = -2;
  }

  // The tile's chunk: which keys exist, whether one has a bad page, and the
  // offsets in the pools: of each eight's first key (WHOLE; the same in all
  // lanes), or of the lane's key in off[0].
  __device__ __forceinline__ uint32_t chunk(const AttendArgs& a, long long (&off)[kSegs], int* bad) const {
    const long long base = head * a.kv.head_stride;
    if (!WHOLE) {
      off[0] = page >= 0 ? page * a.kv.page_stride + base + slot * a.kv.slot_stride : 0;
      *bad = __any_sync(0xffffffffu, page == -2);
      return __ballot_sync(0xffffffffu, page >= 0);
    }
    uint32_t keys = 0;
    *bad = 0;
#pragma unroll
    for (int i = 0; i < kSegs; ++i) {
      const int from = (t - win) * kSegs + i;
      const int pg = __shfl_sync(0xffffffffu, page, from), n = __shfl_sync(0xffffffffu, live, from);
      const int first = __shfl_sync(0xffffffffu, slot, from);
      off[i] = 0;
      if (pg >= 0) {
        off[i] = pg * a.kv.page_stride + base + first * a.kv.slot_stride;
        keys |= ((1u << n) - 1) << (i * kKvSegment);
      }
      *bad |= pg == -2;
    }
    return keys;
  }

  __device__ __forceinline__ StageInfo info(const AttendArgs& a, uint32_t keys, int bad, int block_heads) const {
    return StageInfo{keys, bad, t, tiles, a.pages ? x / a.kv.kv_heads : x, head, u % a.blocks * block_heads, 0};
  }

  // to the next tile, if there is one
  __device__ __forceinline__ void next(const AttendArgs& a) {
    if (--ahead <= 0) return;
    if (++t == tiles) {
      t = 0;
      if (++u == a.units) {
        u = 0;
        win = 1;  // no page that is held belongs to the next entry
        do e = kv_entry(a, ++x);
        while (e.n == 0);
        tiles = kv_tiles(a, e.n);
      }
      head = a.pages ? x % a.kv.kv_heads : u / a.blocks;
    }
    // another unit of the entry goes over the same pages again
    if (!WHOLE || t < win || t - win >= kWindow) look(a);
  }
};

// 16 bytes to shared memory, zeros when `bytes` is 0 (nothing is read then).
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <typename T>
__device__ __forceinline__ T kv_round(float v);
template <>
__device__ __forceinline__ float kv_round<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 kv_round<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }


// What a launch of the attention kernel takes: queries of a group together,
// keys a tile, shared memory of a CTA, CTAs an SM.
struct KernelShape {
  int heads, tile, smem, per_sm;
};
// er_kv_attend_bf16.cu and er_kv_attend_f32.cu: for caches of either type
KernelShape attend_shape_bf16(int d, int group, int q_dtype);
KernelShape attend_shape_f32(int d, int group, int q_dtype);
int attend_bf16(const AttendArgs& a, int q_dtype, cudaStream_t st);
int attend_f32(const AttendArgs& a, int q_dtype, cudaStream_t st);

}  // namespace er
