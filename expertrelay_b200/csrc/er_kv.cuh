// er_kv.cuh -- the paged key-value cache as the er_kv_* kernels see it.
#pragma once

#include <atomic>

#include "er_internal.cuh"

namespace er {

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

// Positions ranked by a score, four at a time: their rank keys in shared
// memory where they fit, else made from the scores each time. In shared
// memory four places behind every 32 stay empty, so that threads which read
// runs of 32 do so from different banks.
struct HeldKeys {
  const uint32_t* held;
  __device__ __forceinline__ static int at(int i) { return i + ((i >> 5) << 2); }
  // keys i .. i + 3, i a multiple of 4 (those behind the last are anything)
  __device__ __forceinline__ uint4 four(int i, int) const { return *reinterpret_cast<const uint4*>(held + at(i)); }
};
inline size_t held_bytes(long long n) { return (size_t)(n + n / 32 * 4 + 40) * 4; }
struct ScoreKeys {
  const float* scores;
  __device__ __forceinline__ uint4 four(int i, int n) const {
    uint4 k = make_uint4(0, 0, 0, 0);
    k.x = rank_key(scores[i]);
    if (i + 1 < n) k.y = rank_key(scores[i + 1]);
    if (i + 2 < n) k.z = rank_key(scores[i + 2]);
    if (i + 3 < n) k.w = rank_key(scores[i + 3]);
    return k;
  }
};

// Bins of one pass of the select: 11, 11, then 10 bits. Shared-memory atomics
// on one address run one by one, and scores crowd into few bins: those of
// exactly zero (sums that nothing was added to yet) are counted a warp at a
// time, and many keys go to four copies of the histogram, by lane.
// Once a bin of few keys is found they are listed and ranked against one another instead.
constexpr int kSelectBins = 2048, kSelectCopies = 4, kSelectMany = 4096, kSelectFew = 512;
inline __host__ __device__ size_t select_bytes(long long most) {  // of the histograms, for at most `most` keys
  return (size_t)kSelectBins * (most >= kSelectMany ? kSelectCopies : 1) * 4;
}

// The `want`-th largest of the keys [lo, hi) of n, by the whole block.
// Returns the threshold; *equal is how many of the keys equal to it belong to
// the `want` largest (the lowest i first). 1 <= want <= hi - lo. `hist`:
// select_bytes(), `red`: one int per warp and four more, shared.
template <typename Keys>
__device__ __forceinline__ uint32_t block_select(const Keys& keys, int n, int lo, int hi, int want, int* hist,
                                                 int* red, int* equal) {
  const int copies = hi - lo >= kSelectMany ? kSelectCopies : 1, warps = blockDim.x >> 5;
  int* mine = hist + (copies > 1 ? (threadIdx.x & (kSelectCopies - 1)) * kSelectBins : 0);
  uint32_t prefix = 0, mask = 0;
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
    for (int b = threadIdx.x; b < copies * kSelectBins; b += blockDim.x) hist[b] = 0;
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
    for (int i = lo / 4 * 4 + (int)threadIdx.x * 4; i < hi; i += blockDim.x * 4) {
      const uint4 k = keys.four(i, n);
      count(k.x, i);
      count(k.y, i + 1);
      count(k.z, i + 2);
      count(k.w, i + 3);
    }
    zeros = __reduce_add_sync(0xffffffffu, zeros);
    if (zeros && (threadIdx.x & 31) == 0) atomicAdd(&mine[(kZeroKey >> shift) & (bins - 1)], zeros);
    __syncthreads();
    // thread t: `per` bins from the top
    const int per = (bins + blockDim.x - 1) / blockDim.x, top = bins - 1 - (int)threadIdx.x * per;
    int sum = 0;
    for (int j = 0; j < per; ++j)
      if (top - j >= 0)
        for (int c = 0; c < copies; ++c) sum += hist[c * kSelectBins + top - j];
    int total;
    int above = block_scan(sum, red, &total);
    if (above < want && want <= above + sum) {
      for (int j = 0; j < per; ++j) {
        int n = 0;
        for (int c = 0; c < copies; ++c) n += hist[c * kSelectBins + top - j];
        if (above < want && want <= above + n) {
          red[warps] = top - j;
          red[warps + 1] = want - above;
          red[warps + 2] = n;
          red[warps + 3] = 0;
        }
        above += n;
      }
    }
    __syncthreads();
    prefix |= (uint32_t)red[warps] << shift;
    mask |= (uint32_t)(bins - 1) << shift;
    want = red[warps + 1];
    const int few = red[warps + 2];
    if (pass == 2 || few > kSelectFew) continue;
    uint32_t* list = reinterpret_cast<uint32_t*>(hist);
    for (int i0 = lo / 4 * 4; i0 < hi; i0 += blockDim.x * 4) {  // a warp's keys get their places together
      const int i = i0 + (int)threadIdx.x * 4;
      const uint4 k4 = i < hi ? keys.four(i, n) : make_uint4(0, 0, 0, 0);
      const uint32_t k[4] = {k4.x, k4.y, k4.z, k4.w};
      int in = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) in |= ((k[e] & mask) == prefix && i + e >= lo && i + e < hi) << e;
      if (!__any_sync(0xffffffffu, in)) continue;
      int at = __popc(in);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, at, o);
        if ((int)(threadIdx.x & 31) >= o) at += up;
      }
      int first = 0;
      if ((threadIdx.x & 31) == 31) first = atomicAdd(&red[warps + 3], at);
      at += __shfl_sync(0xffffffffu, first, 31) - __popc(in);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if ((in >> e) & 1) list[at++] = k[e];
    }
    __syncthreads();
    for (int i = few + threadIdx.x; i < (few + 3) / 4 * 4; i += blockDim.x) list[i] = 0;  // below all that counts
    __syncthreads();
    for (int i = threadIdx.x; i < few; i += blockDim.x) {
      const uint32_t k = list[i];
      int more = 0, same = 0;
#pragma unroll 4
      for (int j = 0; j < few; j += 4) {
        const uint4 x = *reinterpret_cast<const uint4*>(list + j);
        more += (x.x > k) + (x.y > k) + (x.z > k) + (x.w > k);
        same += (x.x == k) + (x.y == k) + (x.z == k) + (x.w == k);
      }
      if (more < want && want <= more + same) {  // the threshold; its equals write the same
        red[warps] = (int)k;
        red[warps + 1] = want - more;
      }
    }
    __syncthreads();
    *equal = red[warps + 1];
    return (uint32_t)red[warps];
  }
  *equal = want;
  return prefix;
}

}  // namespace er
