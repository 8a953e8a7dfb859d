// er_kv_append.cu -- new tokens into the paged key-value cache, and the
// int8 bounds of its pages.
//
// Append: rotate-half RoPE (runtime/qwen_moe.py:126-138, 255-262) on the q
// and k heads of a token's projection row and the write of k and v into the
// token's page. The angle position * theta^(-2j/d) and its sine and cosine
// are taken in 64 bits and rounded once: in 32 bits the product alone loses
// 2^-24 of the angle, 0.004 rad at position 65536 of the fastest channel.
#include <type_traits>

#include "er_kv.cuh"

namespace er {

struct InvFreq {
  double f[128];
};

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// VEC values, 16 bytes of them or a single one, and as fp32.
template <int VEC, typename T>
struct Vec {
  static_assert(VEC == 1 || VEC * sizeof(T) == 16, "one load");
  uint4 raw;

  __device__ __forceinline__ void load(const T* p) {
    if constexpr (VEC == 1) {
      *reinterpret_cast<T*>(&raw) = *p;
    } else {
      raw = ld_stream_u4(p);
    }
  }
  __device__ __forceinline__ void get(float (&x)[VEC]) const {
#pragma unroll
    for (int e = 0; e < VEC; ++e) x[e] = to_f32(reinterpret_cast<const T*>(&raw)[e]);
  }
};
// VEC values to memory, 16 bytes a store (8 where fewer bytes are all).
template <int VEC, typename T>
__device__ __forceinline__ void store_vec(T* p, const float (&x)[VEC]) {
  if constexpr (VEC == 1) {
    *p = from_f32<T>(x[0]);
  } else {
    using S = std::conditional_t<VEC * sizeof(T) == 8, uint2, uint4>;
    constexpr int N = sizeof(S) / sizeof(T);
#pragma unroll
    for (int i = 0; i < VEC; i += N) {
      S raw;
      T* v = reinterpret_cast<T*>(&raw);
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] = from_f32<T>(x[i + e]);
      *reinterpret_cast<S*>(p + i) = raw;
    }
  }
}

// TOK tokens a CTA; a thread turns VEC pairs (j, j + d/2) of a head, or copies
// two VECs of a v head, for each of them. The products and sums of the
// rotation are rounded one by one (no fused multiply-add), so a key's bits do
// not depend on which half of the pair it is, and the pages' codes follow
// from the formula alone. Memory-bound, if enough is in flight: every thread
// has its values of all TOK tokens under way, 16 bytes a load, before the
// angles' sines (64 bits) are computed, by TOK d/2 threads at once. One token a
// CTA while that leaves SMs without work (a decode step), 4 for prompts
// (16384 tokens of 16 + 16 + 16 heads of 128, bf16: 98 us with one, 70). Up to
// 448 threads, so that two CTAs of 72 registers a thread share an SM, in rounds
// of equal size (6745 tokens of 64 + 8 + 8 heads of 96, fp32: 81 us with up to
// 512 threads, 69, where a copy takes 64; loads of 32 bytes a thread: 105).
constexpr int kAppendThreads = 448;

template <typename TX, typename TQ, typename TC, int VEC, int TOK>
__global__ void __launch_bounds__(kAppendThreads, 2)
    kv_append_kernel(KvView kv, const TX* __restrict__ qkv, long long ld, const int32_t* __restrict__ seqs,
                     const int32_t* __restrict__ positions, const int32_t* __restrict__ slots, int n, int heads,
                     const __grid_constant__ InvFreq inv, TQ* __restrict__ q_out, int* status) {
  __shared__ __align__(16) float cs[TOK][256];  // [d/2] cos, then [d/2] sin
  __shared__ long long slot[TOK];               // byte offset of the token's slot in the pools, -1: not written
  kv_enter();
  const int t0 = blockIdx.x * TOK, live = TOK == 1 ? 1 : min(TOK, n - t0);
  const int d = kv.d, half = d / 2, kvh = kv.kv_heads;
  const TX* row = qkv + (long long)t0 * ld;
  const int per = half / VEC, tasks = (heads + 2 * kvh) * per;
  Vec<VEC, TX> va[TOK], vb[TOK];
  auto fetch = [&](int head, int j) {
#pragma unroll
    for (int k = 0; k < TOK; ++k)
      if (k < live) {
        va[k].load(row + k * ld + (long long)head * d + j);
        vb[k].load(row + k * ld + (long long)head * d + j + half);
      }
  };
  int i = threadIdx.x, head = i / per, j = i % per * VEC;
  if (i < tasks) fetch(head, j);
  if ((int)threadIdx.x < live) {
    const int t = t0 + threadIdx.x, pos = slots ? slots[t] : positions[t], seq = seqs ? seqs[t] : t;
    long long off = -1;
    int bad = 0;
    if (seq < 0 || seq >= kv.seqs) {
      bad = ER_KV_BAD_SEQ;
    } else if (pos < 0 || pos >= kv.capacity()) {
      bad = ER_KV_BAD_LENGTH;
    } else {
      const int page = kv.pages_of(seq)[kv.ordinal(pos)];
      if (page < 0 || page >= kv.num_pages)
        bad = ER_KV_BAD_PAGE;
      else
        off = page * kv.page_stride + kv.slot(pos) * kv.slot_stride;
    }
    slot[threadIdx.x] = off;
    if (bad) kv_report(status, bad);
  }
#pragma unroll 1
  for (int f = threadIdx.x; f < live * half; f += blockDim.x) {
    const int k = f / half, c0 = f - k * half;
    double s, c;
    sincos((double)positions[t0 + k] * inv.f[c0], &s, &c);
    cs[k][c0] = (float)c;
    cs[k][half + c0] = (float)s;
  }
  __syncthreads();
#pragma unroll 1
  while (i < tasks) {
#pragma unroll
    for (int k = 0; k < TOK; ++k) {
      if (k >= live) break;
      float a[VEC], b[VEC];
      va[k].get(a);
      vb[k].get(b);
      if (head < heads + kvh) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float c = cs[k][j + e], s = cs[k][half + j + e], x = a[e], y = b[e];
          a[e] = __fsub_rn(__fmul_rn(x, c), __fmul_rn(y, s));
          b[e] = __fadd_rn(__fmul_rn(y, c), __fmul_rn(x, s));
        }
      }
      if (head < heads) {
        TQ* o = q_out + ((long long)(t0 + k) * heads + head) * d + j;
        store_vec<VEC>(o, a);
        store_vec<VEC>(o + half, b);
      } else if (slot[k] >= 0) {
        const bool key = head < heads + kvh;
        char* pool = key ? kv.k : kv.v;
        const long long h = key ? head - heads : head - heads - kvh;
        TC* o = reinterpret_cast<TC*>(pool + slot[k] + h * kv.head_stride) + j;
        store_vec<VEC>(o, a);
        store_vec<VEC>(o + half, b);
      }
    }
    i += blockDim.x;
    if (i >= tasks) break;
    head = i / per;
    j = i % per * VEC;
    fetch(head, j);
  }
}

// Least and greatest key of every channel of a page, a CTA per (page, key
// head): a warp's lanes split a slot's 16-byte columns, lane groups and warps
// the slots, so that a page's loads are all under way at once (after a decode
// step only one page of a sequence changes). The warps' results meet in
// shared memory. Where a CTA has several pages to do, each warp does its own
// (4096 pages of 64 slots: 20 us, 35 with a CTA a page). COLS: columns a lane (2 for fp32 rows over 512 bytes).
constexpr int kBoundsWarps = 4;

template <typename TC, int COLS>
__global__ void __launch_bounds__(kBoundsWarps * 32)
    kv_bounds_kernel(KvView kv, const int32_t* __restrict__ lens, const int32_t* __restrict__ start,
                     int8_t* __restrict__ codes, float* __restrict__ scales, int* status) {
  constexpr int V = 16 / sizeof(TC);
  __shared__ __align__(16) float low[kBoundsWarps][COLS * 32 * V], high[kBoundsWarps][COLS * 32 * V];
  kv_enter();
  const int seq = blockIdx.y, h = blockIdx.z, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int len = lens[seq], from = start[seq], ps = kv.page_size, d = kv.d;
  if (len < 0 || len > kv.capacity() || from < 0) {
    if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0) kv_report(status, ER_KV_BAD_LENGTH);
    return;
  }
  if (from >= len) return;
  const int cols = d / V;  // 1 .. 64
  int wide = 1;            // lanes across a slot
  while (wide < cols && wide < 32) wide *= 2;
  const int first = from / ps, last = (len - 1) / ps;
  const bool solo = last - first >= (int)gridDim.x;  // the same for the whole CTA
  const int each = solo ? kBoundsWarps : 1, mine = solo ? 0 : warp;
  const int col = lane % wide, group = mine * (32 / wide) + lane / wide;
  const int groups = (solo ? 1 : kBoundsWarps) * (32 / wide);
#pragma unroll 1
  for (int o = first + blockIdx.x * each + (solo ? warp : 0); o <= last; o += gridDim.x * each) {
    const int page = kv.pages_of(seq)[o];
    if (page < 0 || page >= kv.num_pages) {
      if (lane == 0) kv_report(status, ER_KV_BAD_PAGE);
      continue;
    }
    const int slots = min(ps, len - o * ps);
    const char* base = kv.k + page * kv.page_stride + h * kv.head_stride;
    float lo[COLS][V], hi[COLS][V], top = 0.f;
#pragma unroll
    for (int w = 0; w < COLS; ++w) {
#pragma unroll
      for (int e = 0; e < V; ++e) lo[w][e] = INFINITY, hi[w][e] = -INFINITY;
      const int c = col + 32 * w;
      if (c < cols) {
#pragma unroll 8
        for (int s = group; s < slots; s += groups) {
          const uint4 raw = *reinterpret_cast<const uint4*>(base + s * kv.slot_stride + c * 16);
          const TC* x = reinterpret_cast<const TC*>(&raw);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float f = to_f32(x[e]);
            lo[w][e] = fminf(lo[w][e], f);
            hi[w][e] = fmaxf(hi[w][e], f);
          }
        }
      }
#pragma unroll 1
      for (int x = wide; x < 32; x *= 2) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          lo[w][e] = fminf(lo[w][e], __shfl_xor_sync(0xffffffffu, lo[w][e], x));
          hi[w][e] = fmaxf(hi[w][e], __shfl_xor_sync(0xffffffffu, hi[w][e], x));
        }
      }
      if (!solo && lane < wide && c < cols) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          low[warp][c * V + e] = lo[w][e];
          high[warp][c * V + e] = hi[w][e];
        }
      }
    }
    if (!solo) __syncthreads();
    // every warp joins all channels (for the scale); lane l has columns l and l + 32
#pragma unroll
    for (int w = 0; w < COLS; ++w) {
      const int c = lane + 32 * w;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if (!solo) lo[w][e] = INFINITY, hi[w][e] = -INFINITY;
        if (c < cols) {
#pragma unroll
          for (int k = 0; k < (solo ? 0 : kBoundsWarps); ++k) {
            lo[w][e] = fminf(lo[w][e], low[k][c * V + e]);
            hi[w][e] = fmaxf(hi[w][e], high[k][c * V + e]);
          }
          if (lo[w][e] <= hi[w][e]) top = fmaxf(top, fmaxf(fabsf(lo[w][e]), fabsf(hi[w][e])));
        }
      }
    }
    if (!solo) __syncthreads();  // the page after this one may be written
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    const float scale = top * kCodeStep;
    const long long at = ((long long)page * kv.kv_heads + h) * 2 * d;
    if (lane == 0 && mine == 0) scales[(long long)page * kv.kv_heads + h] = scale;
    auto code = [&](float x) {  // 0 where there is no number; a division each, as the codes are defined
      const float r = rintf(x / scale);
      return r == r ? (int)fminf(fmaxf(r, -127.f), 127.f) : 0;
    };
#pragma unroll
    for (int w = 0; w < COLS; ++w) {
      const int c = lane + 32 * w;
      if (c >= cols) break;
#pragma unroll
      for (int e = 0; e < V; e += 4) {
        if (!solo && (V == 8 ? e / 4 != warp : warp > 0)) continue;  // four channels a lane and warp
        uint32_t a = 0, b = 0;
#pragma unroll
        for (int f = 0; f < 4; ++f) {
          const bool some = scale > 0.f && lo[w][e + f] <= hi[w][e + f];
          a |= (uint32_t)(uint8_t)(some ? code(lo[w][e + f]) : 0) << (8 * f);
          b |= (uint32_t)(uint8_t)(some ? code(hi[w][e + f]) : 0) << (8 * f);
        }
        *reinterpret_cast<uint32_t*>(codes + at + c * V + e) = a;
        *reinterpret_cast<uint32_t*>(codes + at + d + c * V + e) = b;
      }
    }
  }
}

namespace {

// theta^(-2j/d), kept for the last (theta, d) of the calling thread
const InvFreq& inv_freq(double theta, int d) {
  static thread_local InvFreq f;
  static thread_local double last_theta = 0.0;
  static thread_local int last_d = 0;
  if (theta != last_theta || d != last_d) {
    for (int j = 0; j < d / 2; ++j) f.f[j] = pow(theta, -2.0 * j / d);
    last_theta = theta;
    last_d = d;
  }
  return f;
}

template <typename TX, typename TQ, typename TC>
int append_go(const KvView& kv, const void* qkv, long long ld, const int32_t* seqs, const int32_t* positions,
              const int32_t* slots, int n, int heads, double theta, void* q_out, int* status, cudaStream_t st) {
  // wide accesses need half a head in whole VECs and aligned rows
  constexpr int V = 16 / sizeof(TX);
  const bool vec = kv.d % 16 == 0 && !(((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)(ld * sizeof(TX))) & 15);
  const int tasks = (heads + 2 * kv.kv_heads) * (kv.d / 2) / (vec ? V : 1);  // of a token
  const int rounds = (tasks + kAppendThreads - 1) / kAppendThreads, threads = (tasks + 32 * rounds - 1) / (32 * rounds) * 32;
  const bool many = vec && n >= 148 * 8;
  return launch_chained(!vec   ? kv_append_kernel<TX, TQ, TC, 1, 1>
                        : many ? kv_append_kernel<TX, TQ, TC, V, 4>
                               : kv_append_kernel<TX, TQ, TC, V, 1>,
                        dim3(many ? (n + 3) / 4 : n), dim3(threads), 0, st, "kv_append_kernel", kv, (const TX*)qkv, ld,
                        seqs, positions, slots, n, heads, inv_freq(theta, kv.d), (TQ*)q_out, status);
}

}  // namespace
}  // namespace er

using namespace er;

extern "C" int er_kv_append(const er_kv_cache* cache, const void* qkv, int qkv_dtype, long long ld,
                            const int32_t* seqs, const int32_t* positions, const int32_t* slots, int n, int heads,
                            double theta, void* q_out, int q_dtype, int* status, void* stream) {
  if (int rc = kv_check("er_kv_append", cache)) return rc;
  if (n < 0 || heads <= 0 || heads > kMaxHeads || !(theta > 0))
    return fail(ER_EINVAL, "er_kv_append: n %d, heads %d, theta %g", n, heads, theta);
  if ((qkv_dtype != ER_DTYPE_F32 && qkv_dtype != ER_DTYPE_BF16) || (q_dtype != ER_DTYPE_F32 && q_dtype != ER_DTYPE_BF16))
    return fail(ER_EINVAL, "er_kv_append: dtypes %d, %d", qkv_dtype, q_dtype);
  if (ld < (long long)(heads + 2 * cache->kv_heads) * cache->head_dim)
    return fail(ER_EINVAL, "er_kv_append: row stride %lld shorter than q|k|v (%lld)", ld,
                (long long)(heads + 2 * cache->kv_heads) * cache->head_dim);
  if (n == 0) return ER_OK;
  if (!qkv || !positions || !q_out) return fail(ER_EINVAL, "er_kv_append: null pointer");
  const KvView kv = kv_view(*cache);
  cudaStream_t st = (cudaStream_t)stream;
  const int sel = (qkv_dtype == ER_DTYPE_BF16) * 4 + (q_dtype == ER_DTYPE_BF16) * 2 + (cache->dtype == ER_DTYPE_BF16);
  using bf = __nv_bfloat16;
  switch (sel) {
    case 0: return append_go<float, float, float>(kv, qkv, ld, seqs, positions, slots, n, heads, theta, q_out, status, st);
    case 1: return append_go<float, float, bf>(kv, qkv, ld, seqs, positions, slots, n, heads, theta, q_out, status, st);
    case 2: return append_go<float, bf, float>(kv, qkv, ld, seqs, positions, slots, n, heads, theta, q_out, status, st);
    case 3: return append_go<float, bf, bf>(kv, qkv, ld, seqs, positions, slots, n, heads, theta, q_out, status, st);
    case 4: return append_go<bf, float, float>(kv, qkv, ld, seqs, positions, slots, n, heads, theta, q_out, status, st);
    case 5: return append_go<bf, float, bf>(kv, qkv, ld, seqs, positions, slots, n, heads, theta, q_out, status, st);
    case 6: return append_go<bf, bf, float>(kv, qkv, ld, seqs, positions, slots, n, heads, theta, q_out, status, st);
    default: return append_go<bf, bf, bf>(kv, qkv, ld, seqs, positions, slots, n, heads, theta, q_out, status, st);
  }
}

extern "C" int er_kv_page_bounds(const er_kv_cache* cache, const int32_t* lens, const int32_t* start, int8_t* codes,
                                 float* scales, int* status, void* stream) {
  if (int rc = kv_check("er_kv_page_bounds", cache)) return rc;
  if (cache->seqs == 0 || cache->table_width == 0) return ER_OK;
  if (!lens || !start || !codes || !scales) return fail(ER_EINVAL, "er_kv_page_bounds: null pointer");
  if ((uintptr_t)codes & 7) return fail(ER_EINVAL, "er_kv_page_bounds: codes must be 8-byte aligned");
  if (cache->seqs > 65535) return fail(ER_EINVAL, "er_kv_page_bounds: %d sequences (at most 65535)", cache->seqs);
  const KvView kv = kv_view(*cache);
  // a step touches one page a sequence, a prompt all of them: the CTAs of a
  // (sequence, key head) walk its pages, about 16 CTAs an SM in all
  const long long want = 148 * 16 / ((long long)kv.seqs * kv.kv_heads), most = kv.width;
  const unsigned gx = (unsigned)(want < 1 ? 1 : want > most ? most : want);
  const dim3 grid(gx, kv.seqs, kv.kv_heads);
  return launch_chained(cache->dtype == ER_DTYPE_BF16 ? kv_bounds_kernel<__nv_bfloat16, 1>
                        : kv.d > 128                  ? kv_bounds_kernel<float, 2>
                                                      : kv_bounds_kernel<float, 1>,
                        grid, dim3(128), 0, (cudaStream_t)stream, "kv_bounds_kernel", kv, lens, start, codes, scales,
                        status);
}
