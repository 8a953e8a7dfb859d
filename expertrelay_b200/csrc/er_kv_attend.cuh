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
constexpr int kKvChunk = 16;  // keys a warp takes at a time

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
  int tile;                    // keys a tile: warps a CTA * kKvChunk
  int shift;                   // log2 of page_size, -1 when it is no power of two
  int min_share;               // the least share of the line worth a CTA
  int* status;
  // scan entries: rows, or (row, key head) pairs when each has its own page list
  int entries, units;          // units of one entry: the tiles repeat that often
  CutUnit* cut;                // [grid] the unit that begins in a CTA's run and ends behind it
  float* part_ml;              // [2 grid][GB][2]: m, l of a CTA's first and last piece
  float* part_o;               // [2 grid][GB][d]
  int grid;                    // CTAs of the attention kernel
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

static __device__ __noinline__ Entry kv_entry(const AttendArgs& a, int x) {
  const int row = a.pages ? x / a.kv.kv_heads : x;
  Entry e;
  e.seq = a.seqs ? a.seqs[row] : row;
  e.len = a.lens[row];
  e.n = e.len;
  e.bad = 0;
  if (e.seq < 0 || e.seq >= a.kv.seqs) {
    e.bad = ER_KV_BAD_SEQ;
  } else if (e.len < 0 || e.len > kKvMaxLen || e.len > a.kv.capacity() || (a.scores && e.len > a.mass_len)) {
    e.bad = ER_KV_BAD_LENGTH;
  } else if (a.pages) {
    const int c = a.counts[x];
    if (c < 0 || c > a.max_pages || (long long)c * a.kv.page_size > kKvMaxLen)
      e.bad = ER_KV_BAD_LENGTH;
    else
      e.n = c * a.kv.page_size;  // positions behind len are left out key by key
  }
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

// 64-bit division as a call: inlined, each is a hundred instructions that
// a short launch would fetch for the first time.
static __device__ __noinline__ long long kv_div(long long a, long long b) { return a / b; }
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

// A tile: entry x, unit u of it, tile t of that unit's.
struct Place {
  int x, u, t, tiles, head;  // head: key head
  Entry e;

  __device__ __forceinline__ void set(const AttendArgs& a, int entry, int unit, int tile) {
    x = entry;
    u = unit;
    t = tile;
    e = kv_entry(a, x);
    tiles = kv_tiles(a, e.n);
    head = a.pages ? x % a.kv.kv_heads : u / a.blocks;
  }
  // The next tile; the caller knows that there is one.
  __device__ __forceinline__ void next(const AttendArgs& a) {
    if (++t < tiles) return;
    int y = x, v = u + 1;
    if (v == a.units) {
      v = 0;
      do ++y;
      while (kv_entry(a, y).n == 0);
    }
    set(a, y, v, 0);
  }
  __device__ __forceinline__ int row(const AttendArgs& a) const { return a.pages ? x / a.kv.kv_heads : x; }
  __device__ __forceinline__ int block(const AttendArgs& a) const { return u % a.blocks; }  // head block of the group
};

// What a CTA works through: `left` tiles from a place on; `begin` is where
// the first tile's unit begins in the line of length `total`.
struct Run {
  long long left, begin, total;
};

// Every CTA sums the entries' costs itself (a few loads a thread) and finds
// its share's ends. `sums`: 2 (blockDim.x + 1) long longs, `where`: 3 ints,
// `ends`: 3 long longs, shared.
__device__ __forceinline__ Run kv_run(const AttendArgs& a, long long* sums, int* where, long long* ends, Place& p) {
  const int threads = blockDim.x;
  if (threadIdx.x == 0) {
    a.cut[blockIdx.x].row = -1;
    sums[0] = sums[threads + 1] = 0;
  }
  const int per = (a.entries + threads - 1) / threads;
  const int x0 = min(a.entries, (int)threadIdx.x * per), x1 = min(a.entries, x0 + per);
  long long cost = 0, tiles = 0;
#pragma unroll 1
  for (int x = x0; x < x1; ++x) {
    const Entry e = kv_entry(a, x);
    const int c = kv_tiles(a, e.n);
    tiles += c;
    cost += kv_cost(c);
    if (blockIdx.x == 0 && e.bad) kv_report(a.status, e.bad);
  }
  long long* tsum = sums + threads + 1;
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long uc = __shfl_up_sync(0xffffffffu, cost, o), ut = __shfl_up_sync(0xffffffffu, tiles, o);
    if (lane >= o) {
      cost += uc;
      tiles += ut;
    }
  }
  sums[threadIdx.x + 1] = cost;
  tsum[threadIdx.x + 1] = tiles;
  __syncthreads();
  long long c0 = 0, t0 = 0, all = 0, all_tiles = 0;  // before this warp, and in all
#pragma unroll 1
  for (int w = 1; w <= threads / 32; ++w) {
    if (w == (int)threadIdx.x / 32 + 1) {
      c0 = all;
      t0 = all_tiles;
    }
    all += sums[w * 32];
    all_tiles += tsum[w * 32];
  }
  const long long total = all * a.units;
  if (total == 0) return Run{0, 0, 0};
  const int shares = kv_shares(a, total);
  if ((int)blockIdx.x >= shares) return Run{0, 0, total};
  // this thread's entries: the line from ex on, `tb` tiles before it
  const long long ex = (c0 + (lane ? sums[threadIdx.x] : 0)) * a.units, in = (c0 + cost) * a.units;
  const long long tb = (t0 + (lane ? tsum[threadIdx.x] : 0)) * a.units;
#pragma unroll 1
  for (int end = 0; end < 2; ++end) {
    const long long at = kv_share_start(total, shares, blockIdx.x + end);
    if (at == total && threadIdx.x == 0) ends[1] = all_tiles * a.units;
    if (at < ex || at >= in) continue;
    long long rest = at - ex, before = tb;
#pragma unroll 1
    for (int x = x0; x < x1; ++x) {
      const int c = kv_tiles(a, kv_entry(a, x).n), k = kv_cost(c);
      if (rest < (long long)k * a.units) {
        const int u = (int)kv_div(rest, k), in_unit = (int)(rest - (long long)u * k), t = max(0, in_unit - kUnitCost);
        ends[end] = before + (long long)u * c + t;
        if (end == 0) {
          where[0] = x;
          where[1] = u;
          where[2] = t;
          ends[2] = at - in_unit;
        }
        break;
      }
      rest -= (long long)k * a.units;
      before += (long long)c * a.units;
    }
  }
  __syncthreads();
  p.set(a, where[0], where[1], where[2]);
  return Run{ends[1] - ends[0], ends[2], total};
}

// Where key j of a place lies: byte offset of its slot in the pools, or -1
// when there is no such key (behind the length, a list's page behind it) and
// -2 when its page id is bad.
__device__ __forceinline__ long long kv_locate(const AttendArgs& a, const Place& p, int j) {
  if (j >= p.e.n) return -1;
  int o = a.shift >= 0 ? j >> a.shift : j / a.kv.page_size;
  const int slot = j - o * a.kv.page_size;
  if (a.pages) {
    o = a.pages[(long long)p.x * a.max_pages + o];
    if (o < 0 || o >= a.kv.width) return -2;
    if ((long long)o * a.kv.page_size + slot >= p.e.len) return -1;
  }
  const int page = a.kv.pages_of(p.e.seq)[o];
  if (page < 0 || page >= a.kv.num_pages) return -2;
  return page * a.kv.page_stride + p.head * a.kv.head_stride + slot * a.kv.slot_stride;
}

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

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

// 2^(m_i - m) of a piece, 0 for a piece without keys or of -inf scores alone.
__device__ __forceinline__ float piece_weight(float mi, float m) { return mi == -INFINITY ? 0.f : exp2f(mi - m); }


// What a launch of an attention kernel takes: queries of a group together,
// warps and shared memory of a CTA, CTAs an SM.
struct KernelShape {
  int heads, warps, smem, per_sm;
};
// the tensor-core kernel for bf16 caches (er_kv_attend_mma.cu)
KernelShape mma_shape(int d, int group, int q_dtype);
int attend_mma(const AttendArgs& a, int q_dtype, cudaStream_t st);

}  // namespace er
