// er_kv.cuh -- the paged key-value cache as the er_kv_* kernels see it.
#pragma once

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

  __device__ __forceinline__ const int32_t* pages_of(int seq) const { return table + (long long)seq * table_stride; }
  // positions the table has room for (64 bits: width * page_size may pass 2^31)
  __device__ __forceinline__ long long capacity() const { return (long long)width * page_size; }
};

inline KvView kv_view(const er_kv_cache& c) {
  const long long es = c.dtype == ER_DTYPE_BF16 ? 2 : 4;
  return KvView{(char*)c.k,     (char*)c.v,  c.page_stride * es, c.head_stride * es, c.slot_stride * es, c.table,
                c.table_stride, c.num_pages, c.page_size,        c.kv_heads,         c.head_dim,         c.seqs,
                c.table_width};
}

inline int kv_check(const char* who, const er_kv_cache* c) {
  if (!c) return fail(ER_EINVAL, "%s: null cache", who);
  if (c->dtype != ER_DTYPE_F32 && c->dtype != ER_DTYPE_BF16) return fail(ER_EINVAL, "%s: cache dtype %d", who, c->dtype);
  if (c->num_pages <= 0 || c->page_size <= 0 || c->kv_heads <= 0 || c->seqs < 0 || c->table_width < 0)
    return fail(ER_EINVAL, "%s: %d pages of %d positions, %d key heads, table of %d x %d", who, c->num_pages,
                c->page_size, c->kv_heads, c->seqs, c->table_width);
  if (c->head_dim <= 0 || c->head_dim % 8 || c->head_dim > 256)
    return fail(ER_EINVAL, "%s: head_dim %d (a multiple of 8, at most 256)", who, c->head_dim);
  if (!c->k || !c->v || (c->seqs > 0 && c->table_width > 0 && !c->table)) return fail(ER_EINVAL, "%s: null pointer", who);
  const long long es = c->dtype == ER_DTYPE_BF16 ? 2 : 4;
  if (((uintptr_t)c->k | (uintptr_t)c->v | (uintptr_t)(c->page_stride * es) | (uintptr_t)(c->head_stride * es) |
       (uintptr_t)(c->slot_stride * es)) & 15)
    return fail(ER_EINVAL, "%s: slots must lie on 16-byte boundaries", who);
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
  int before = 0, all = 0;
  for (int w = 0; w < warps; ++w) {
    if (w < warp) before += red[w];
    all += red[w];
  }
  *total = all;
  return before + inc - v;
}

// The `want`-th largest of key(i), i in [lo, hi), by the whole block: 8 bits
// a pass from the top. Returns the threshold; *equal is how many of the keys
// equal to it belong to the `want` largest (the lowest i first). want >= 1,
// want <= hi - lo. `hist`: 256 ints, `red`: 2 ints, shared.
template <typename Key>
__device__ uint32_t block_select(Key key, int lo, int hi, int want, int* hist, int* red, int* equal) {
  uint32_t prefix = 0, mask = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int b = threadIdx.x; b < 256; b += blockDim.x) hist[b] = 0;
    __syncthreads();
    for (int i = lo + (int)threadIdx.x; i < hi; i += blockDim.x) {
      const uint32_t k = key(i);
      if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1);
    }
    __syncthreads();
    if (threadIdx.x < 32) {  // lane l: bins 255 - 8 l .. 248 - 8 l, from the top
      int c[8], sum = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += c[j] = hist[255 - 8 * (int)threadIdx.x - j];
      int inc = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, inc, o);
        if ((int)threadIdx.x >= o) inc += up;
      }
      int above = inc - sum;
      if (above < want && want <= inc) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (above < want && want <= above + c[j]) {
            red[0] = 255 - 8 * (int)threadIdx.x - j;
            red[1] = want - above;
          }
          above += c[j];
        }
      }
    }
    __syncthreads();
    prefix |= (uint32_t)red[0] << shift;
    mask |= 255u << shift;
    want = red[1];
  }
  *equal = want;
  return prefix;
}

}  // namespace er
