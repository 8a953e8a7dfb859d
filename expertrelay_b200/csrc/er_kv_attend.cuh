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
  long long begin, total;  // its first tile, and all tiles of the launch
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
  int min_tiles;               // fewest tiles worth a CTA
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

__device__ __forceinline__ Entry kv_entry(const AttendArgs& a, int x) {
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

// CTAs that share `total` tiles, the first tile of CTA i, and the CTA that has tile x.
__device__ __forceinline__ int kv_shares(const AttendArgs& a, long long total) {
  const long long s = (total + a.min_tiles - 1) / a.min_tiles;
  return (int)(s < a.grid ? s : a.grid);
}
__device__ __forceinline__ long long kv_share_start(long long total, int shares, int i) { return total * i / shares; }
__device__ __forceinline__ int kv_share_of(long long total, int shares, long long x) {
  return (int)(((x + 1) * shares - 1) / total);
}

// A place in the line of tiles: entry x, unit u of it, tile t of that unit.
struct Place {
  int x, u, t, tiles;
  Entry e;

  __device__ __forceinline__ void load(const AttendArgs& a, int entry) {
    x = entry;
    e = kv_entry(a, x);
    tiles = kv_tiles(a, e.n);
  }
  // The next tile; the caller knows that there is one.
  __device__ __forceinline__ void next(const AttendArgs& a) {
    if (++t < tiles) return;
    t = 0;
    if (++u < a.units) return;
    u = 0;
    do load(a, x + 1);
    while (tiles == 0);
  }
  __device__ __forceinline__ int row(const AttendArgs& a) const { return a.pages ? x / a.kv.kv_heads : x; }
  __device__ __forceinline__ int head(const AttendArgs& a) const {  // key head
    return a.pages ? x % a.kv.kv_heads : u / a.blocks;
  }
  __device__ __forceinline__ int block(const AttendArgs& a) const { return u % a.blocks; }  // head block of the group
};

// The CTA's run of tiles: its first place and how many tiles it has. Every
// CTA sums the entries' tiles itself (a few loads a thread). `sums`: blockDim.x + 1 long longs, shared.
struct Run {
  long long begin, left, total;
};
__device__ __forceinline__ Run kv_run(const AttendArgs& a, long long* sums, int* where, Place& p) {
  if (threadIdx.x == 0) a.cut[blockIdx.x].row = -1;
  const int per = (a.entries + blockDim.x - 1) / blockDim.x;
  const int x0 = min(a.entries, (int)threadIdx.x * per), x1 = min(a.entries, x0 + per);
  long long mine = 0;
  for (int x = x0; x < x1; ++x) {
    const Entry e = kv_entry(a, x);
    mine += kv_tiles(a, e.n);
    if (blockIdx.x == 0 && e.bad) kv_report(a.status, e.bad);
  }
  sums[threadIdx.x + 1] = mine;
  if (threadIdx.x == 0) sums[0] = 0;
  __syncthreads();
  if (threadIdx.x < 32) {
    const int each = blockDim.x / 32, l = threadIdx.x;
    long long s = 0;
    for (int i = 0; i < each; ++i) s += sums[1 + l * each + i];
    long long inc = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, inc, o);
      if (l >= o) inc += up;
    }
    long long run = inc - s;
    for (int i = 0; i < each; ++i) {
      run += sums[1 + l * each + i];
      sums[1 + l * each + i] = run;
    }
  }
  __syncthreads();
  const long long per_unit = sums[blockDim.x], total = per_unit * a.units;
  if (total == 0) return Run{0, 0, 0};
  const int shares = kv_shares(a, total);
  if ((int)blockIdx.x >= shares) return Run{0, 0, total};
  const long long begin = kv_share_start(total, shares, blockIdx.x);
  const long long end = kv_share_start(total, shares, blockIdx.x + 1);
  // the entry whose units hold tile `begin`: all units of the entries before it are passed
  const long long ex = sums[threadIdx.x] * a.units, in = sums[threadIdx.x + 1] * a.units;
  if (ex <= begin && begin < in) {
    long long rest = begin - ex;
    for (int x = x0; x < x1; ++x) {
      const long long c = kv_tiles(a, kv_entry(a, x).n);
      if (rest < c * a.units) {
        where[0] = x;
        where[1] = (int)(rest / c);
        where[2] = (int)(rest % c);
        break;
      }
      rest -= c * a.units;
    }
  }
  __syncthreads();
  p.load(a, where[0]);
  p.u = where[1];
  p.t = where[2];
  return Run{begin, end - begin, total};
}

// Where key j of a place lies: byte offset of its slot (key head included)
// in the pools, or -1 when there is no such key (behind the length, a list's
// page behind it) and -2 when its page id is bad.
__device__ __forceinline__ long long kv_locate(const AttendArgs& a, const Place& p, int h, int j) {
  if (j >= p.e.n) return -1;
  const int ps = a.kv.page_size;
  int o = j / ps;
  const int slot = j - o * ps;
  if (a.pages) {
    o = a.pages[(long long)p.x * a.max_pages + o];
    if (o < 0 || o >= a.kv.width) return -2;
    if ((long long)o * ps + slot >= p.e.len) return -1;
  }
  const int page = a.kv.pages_of(p.e.seq)[o];
  if (page < 0 || page >= a.kv.num_pages) return -2;
  return page * a.kv.page_stride + h * a.kv.head_stride + slot * a.kv.slot_stride;
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
