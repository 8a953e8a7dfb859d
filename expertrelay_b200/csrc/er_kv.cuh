// er_kv.cuh -- the paged key-value cache as the er_kv_* kernels see it.
#pragma once

#include <atomic>

#include "er_internal.cuh"

namespace er {

constexpr int kMaxHeads = 65536;  // of queries: their products with head_dim stay ints

// er_kv_cache with strides in bytes (the pools' element type is a template
// parameter of the kernels that touch values).
struct KvView {
  char *k, *v;
  long long page_stride, head_stride, slot_stride;  // bytes
  const int32_t* table;
  long long table_stride;
  int num_pages, page_size, kv_heads, d, seqs, width;
  int shift;  // log2 of page_size, -1 when it is no power of two

  __device__ __forceinline__ const int32_t* pages_of(int seq) const { return table + (long long)seq * table_stride; }
  // the ordinal of the page that holds a position, and the position's slot in it
  __device__ __forceinline__ int ordinal(int pos) const { return shift >= 0 ? pos >> shift : pos / page_size; }
  __device__ __forceinline__ int slot(int pos) const { return shift >= 0 ? pos & (page_size - 1) : pos % page_size; }
  // positions the table has room for (64 bits: width * page_size may pass 2^31)
  __device__ __forceinline__ long long capacity() const { return (long long)width * page_size; }
};

inline KvView kv_view(const er_kv_cache& c) {
  const long long es = c.dtype == ER_DTYPE_BF16 ? 2 : 4;
  int shift = -1;
  for (int b = 0; b < 31; ++b)
    if (c.page_size == 1 << b) shift = b;
  return KvView{(char*)c.k,     (char*)c.v,  c.page_stride * es, c.head_stride * es, c.slot_stride * es, c.table,
                c.table_stride, c.num_pages, c.page_size,        c.kv_heads,         c.head_dim,         c.seqs,
                c.table_width,  shift};
}

inline int kv_check(const char* who, const er_kv_cache* c) {
  if (!c) return fail(ER_EINVAL, "%s: null cache", who);
  if (c->dtype != ER_DTYPE_F32 && c->dtype != ER_DTYPE_BF16) return fail(ER_EINVAL, "%s: cache dtype %d", who, c->dtype);
  if (c->num_pages <= 0 || c->page_size <= 0 || c->kv_heads <= 0 || c->seqs < 0 || c->table_width < 0)
    return fail(ER_EINVAL, "%s: %d pages of %d positions, %d key heads, table of %d x %d", who, c->num_pages,
                c->page_size, c->kv_heads, c->seqs, c->table_width);
  if (c->kv_heads > 1024) return fail(ER_EINVAL, "%s: %d key heads (at most 1024)", who, c->kv_heads);
  if (c->head_dim <= 0 || c->head_dim % 8 || c->head_dim > 256)
    return fail(ER_EINVAL, "%s: head_dim %d (a multiple of 8, at most 256)", who, c->head_dim);
  if (!c->k || !c->v || (c->seqs > 0 && c->table_width > 0 && !c->table)) return fail(ER_EINVAL, "%s: null pointer", who);
  const long long es = c->dtype == ER_DTYPE_BF16 ? 2 : 4;
  if (((uintptr_t)c->k | (uintptr_t)c->v | (uintptr_t)(c->page_stride * es) | (uintptr_t)(c->head_stride * es) |
       (uintptr_t)(c->slot_stride * es)) & 15)
    return fail(ER_EINVAL, "%s: slots must lie on 16-byte boundaries", who);
  return ER_OK;
}

// The current device, and its SMs (asked once a device).
inline int device_sms(int* sms) {
  static std::atomic<int> known[64];
  int dev = 0;
  if (int rc = cuda_check(cudaGetDevice(&dev), "cudaGetDevice")) return rc;
  if (dev < 64 && (*sms = known[dev].load(std::memory_order_relaxed)) > 0) return ER_OK;
  if (int rc = cuda_check(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev), "cudaDeviceGetAttribute"))
    return rc;
  if (dev < 64) known[dev].store(*sms, std::memory_order_relaxed);
  return ER_OK;
}

// Lets `kernel` take up to `bytes` of dynamic shared memory (set once a
// device; `done`: one word per kernel, a bit per device).
template <typename K>
inline int allow_smem(K kernel, int bytes, std::atomic<unsigned long long>& done) {
  int dev = 0;
  if (int rc = cuda_check(cudaGetDevice(&dev), "cudaGetDevice")) return rc;
  const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return ER_OK;
  if (int rc = cuda_check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes),
                          "shared memory attribute"))
    return rc;
  done.fetch_or(bit, std::memory_order_relaxed);
  return ER_OK;
}

__device__ __forceinline__ void kv_report(int* status, int bit) {
  if (status) atomicOr(status, bit);
}

// The step of int8 codes is the greatest magnitude times 1/127 (rounded to 32 bits).
constexpr float kCodeStep = 1.0f / 127.0f;

// The order in which scores rank as unsigned integers: NaN below everything,
// the two zeros alike.
__device__ __forceinline__ uint32_t rank_key(float f) {
  if (f != f) return 0u;
  const uint32_t b = __float_as_uint(f == 0.f ? 0.f : f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// First thing in every kernel: the next one of the chain may launch and run
// up to here beside this one, and nothing of this one reads or writes memory
// before all that was queued earlier is done.
__device__ __forceinline__ void kv_enter() {
  chain_trigger();
  chain_wait();
}

constexpr int kClusterCtas = 8;  // of the kernels that run a cluster for each of few units

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ int cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return (int)r;
}
// Every thread of every CTA of the cluster arrives and waits; what was written before is seen after.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// the address of `addr` (shared memory) in the cluster's CTA `rank`
__device__ __forceinline__ uint32_t cluster_addr(uint32_t addr, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}

__device__ __forceinline__ float2 cluster_load2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}

// Launch with programmatic stream serialization, in clusters of kClusterCtas when `cluster`.
template <typename... KArgs, typename... Args>
inline int kv_launch(void (*kernel)(KArgs...), dim3 grid, int threads, size_t smem, bool cluster, cudaStream_t st,
                     const char* what, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = kClusterCtas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster ? 2 : 1;
  return cuda_check(cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...), what);
}

constexpr uint32_t kZeroKey = 0x80000000u;  // rank_key(0)

// Exclusive prefix of `v` over the block's threads in thread order, and the
// block's sum in *total. `red`: one int per warp plus one, shared.
__device__ __forceinline__ int block_scan(int v, int* red, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += up;
  }
  __syncthreads();  // `red` is free
  if (lane == 31) red[warp] = inc;
  __syncthreads();
  const int mine = lane < warps ? red[lane] : 0;  // at most 32 warps
  int before = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += up;
  }
  *total = __shfl_sync(0xffffffffu, before, 31);
  return __shfl_sync(0xffffffffu, before - mine, warp) + inc - v;
}

// Positions ranked by a score: rank keys in shared memory, four at a time.
// Four places behind every 32 stay empty, so that threads which read runs of
// 32 do so from different banks.
struct HeldKeys {
  const uint32_t* held;
  __host__ __device__ static constexpr int at(int i) { return i + ((i >> 5) << 2); }
  // keys i .. i + 3, i a multiple of 4 (those behind the last are anything)
  __device__ __forceinline__ uint4 four(int i) const { return *reinterpret_cast<const uint4*>(held + at(i)); }
};
inline size_t held_bytes(long long n) { return (size_t)(n + n / 32 * 4 + 40) * 4; }

// Bins of one pass of the select: 11, 11, then 10 bits. Shared-memory atomics
// on one address run one by one, and scores crowd into few bins: those of
// exactly zero (sums that nothing was added to yet) are counted a thread at a
// time, and many keys go to four copies of the histogram, by lane.
constexpr int kSelectBins = 2048, kSelectCopies = 4, kSelectMany = 4096;
inline __host__ __device__ size_t select_bytes(long long most) {  // of the histograms, for at most `most` keys a CTA
  return (size_t)kSelectBins * (most >= kSelectMany ? kSelectCopies : 1) * 4;
}

// What the CTAs that choose together (a cluster of C, or one alone) share.
struct SelectScratch {
  int red[34];    // block_scan; the bin and the rank in it that a pass finds
  int counts[2];  // this CTA's keys above the threshold, and equal to it
};

// Chooses `take` of n ranked positions, n > take: the first `sinks` and the
// last `recent`, then those of the greatest keys, equal ones from the lowest
// position on; emit(slot, i) for each chosen position i, slots in position
// order. By the C CTAs of a cluster together (rank r holds the keys of the nl
// positions from b0 on, in rank order) or by one (C = 1). A radix select from
// the top bits down finds the least key that is taken: every CTA counts its
// own keys, then sums all CTAs' histograms; last, the CTAs' counts place each
// one's positions. sinks + recent <= take. `hist`: select_bytes(), shared.
template <int C, typename Emit>
__device__ __forceinline__ void take_best(const HeldKeys& keys, int b0, int nl, int n, int take, int sinks, int recent,
                                          int* hist, SelectScratch& sc, Emit emit) {
  const int lo = sinks, hi = n - recent;
  int want = take - sinks - recent;
  const int copies = nl >= kSelectMany ? kSelectCopies : 1;
  const int rank = C > 1 ? cluster_rank() : 0;
  auto meet = [&]() {
    if (C > 1)
      cluster_sync();
    else
      __syncthreads();
  };
  const uint32_t hist0 = smem_addr(hist);
  int* mine = hist + (copies > 1 ? (threadIdx.x & (kSelectCopies - 1)) * kSelectBins : 0);
  uint32_t prefix = 0, mask = 0;
  if (want > 0) {
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
      for (int b = threadIdx.x * 4; b < copies * kSelectBins; b += blockDim.x * 4)
        *reinterpret_cast<int4*>(hist + b) = make_int4(0, 0, 0, 0);
      __syncthreads();
      int zeros = 0;  // of this thread
      auto count = [&](uint32_t k, int i) {
        if ((k & mask) != prefix || i < lo || i >= hi) return;
        if (k == kZeroKey)
          ++zeros;
        else
          atomicAdd(&mine[(k >> shift) & (bins - 1)], 1);
      };
#pragma unroll 2
      for (int i = threadIdx.x * 4; i < nl; i += blockDim.x * 4) {
        const uint4 k = keys.four(i);
        count(k.x, b0 + i);
        if (i + 1 < nl) count(k.y, b0 + i + 1);
        if (i + 2 < nl) count(k.z, b0 + i + 2);
        if (i + 3 < nl) count(k.w, b0 + i + 3);
      }
      zeros = __reduce_add_sync(0xffffffffu, zeros);
      if (zeros && (threadIdx.x & 31) == 0) atomicAdd(&mine[(kZeroKey >> shift) & (bins - 1)], zeros);
      if (copies > 1) {
        __syncthreads();
        for (int b = threadIdx.x; b < bins; b += blockDim.x) {
          int c = hist[b];
          for (int j = 1; j < kSelectCopies; ++j) c += hist[j * kSelectBins + b];
          hist[b] = c;
        }
      }
      meet();
      // four bins a thread, from the top (a block has at least 256 threads, so two rounds at the most)
      int above = 0;
#pragma unroll 1
      for (int top = bins - 4 - (int)threadIdx.x * 4, round = 0; round * (int)blockDim.x * 4 < bins;
           ++round, top -= blockDim.x * 4) {
        int4 c = make_int4(0, 0, 0, 0);
        if (top >= 0) {
#pragma unroll
          for (int r = 0; r < C; ++r) {
            int4 x;
            if (C > 1)
              asm volatile("ld.shared::cluster.v4.u32 {%0,%1,%2,%3}, [%4];"
                           : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                           : "r"(cluster_addr(hist0, r) + top * 4)
                           : "memory");
            else
              x = *reinterpret_cast<const int4*>(hist + top);
            c.x += x.x;
            c.y += x.y;
            c.z += x.z;
            c.w += x.w;
          }
        }
        const int sum = c.x + c.y + c.z + c.w;
        int total;
        int at = above + block_scan(sum, sc.red, &total);
        above += total;
        if (at < want && want <= at + sum) {
          const int n4[4] = {c.w, c.z, c.y, c.x};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (at < want && want <= at + n4[j]) {
              sc.red[32] = top + 3 - j;
              sc.red[33] = want - at;
            }
            at += n4[j];
          }
        }
      }
      meet();  // the bin is found, and the histograms may be written again
      prefix |= (uint32_t)sc.red[32] << shift;
      mask |= (uint32_t)(bins - 1) << shift;
      want = sc.red[33];
    }
  } else {
    want = 0;
  }
  const uint32_t least = prefix;  // `want` of the keys equal to it are taken; without any, none is above or equal
  const bool none = mask == 0;
  // a run of 4, 8, .. 32 positions a thread, in rounds; first how many there are, then where they go
  int run = 4;
  while (run < 32 && run * (int)blockDim.x < nl) run *= 2;
  auto look = [&](int b, uint32_t* sure, uint32_t* tied) {
    *sure = *tied = 0;
    for (int j = 0; j < run && b + j < nl; j += 4) {
      const uint4 k4 = keys.four(b + j);
      const uint32_t k[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = b0 + b + j + e;
        const bool forced = i < lo || i >= hi, there = b + j + e < nl;
        *sure |= (uint32_t)(there && (forced || (!none && k[e] > least))) << (j + e);
        *tied |= (uint32_t)(there && !forced && !none && k[e] == least) << (j + e);
      }
    }
  };
  int above = 0, same = 0;  // taken outright, and equal to the threshold, before this CTA's positions
  if (C > 1) {
    int s = 0, q = 0;
    for (int r0 = 0; r0 < nl; r0 += run * blockDim.x) {
      uint32_t sure, tied;
      look(r0 + (int)threadIdx.x * run, &sure, &tied);
      s += __popc(sure);
      q += __popc(tied);
    }
    int all_s, all_q;
    block_scan(s, sc.red, &all_s);
    block_scan(q, sc.red, &all_q);
    if (threadIdx.x == 0) {
      sc.counts[0] = all_s;
      sc.counts[1] = all_q;
    }
    cluster_sync();
    const uint32_t at = smem_addr(sc.counts);
    for (int r = 0; r < rank; ++r) {
      const float2 c = cluster_load2(cluster_addr(at, r));
      above += __float_as_int(c.x);
      same += __float_as_int(c.y);
    }
  }
  for (int r0 = 0; r0 < nl; r0 += run * blockDim.x) {
    const int b = r0 + (int)threadIdx.x * run;
    uint32_t sure, tied;
    look(b, &sure, &tied);
    // 16 bits each, without sign: a round has at most 32 * 1024 positions
    int all;
    const int before = block_scan(__popc(sure) | __popc(tied) << 16, sc.red, &all);
    int at = above + (before & 0xffff), tie = same + (int)((uint32_t)before >> 16);
    for (uint32_t left = sure | tied; left; left &= left - 1) {
      const int j = __ffs(left) - 1;
      if ((sure >> j) & 1) {
        emit(at + min(tie, want), b0 + b + j);
        ++at;
      } else {
        if (tie < want) emit(at + tie, b0 + b + j);
        ++tie;
      }
    }
    above += all & 0xffff;
    same += (int)((uint32_t)all >> 16);
  }
  meet();  // no CTA leaves while its counts may be read
}

}  // namespace er
