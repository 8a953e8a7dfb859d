// er_kv_select.cu -- the pages worth reading for each query, and the
// positions worth keeping in a cache that grows too long.
//
// Both rank by a score and take the best (take_best in er_kv.cuh): equal
// scores to the lower position, the taken ones in position order.
#include "er_kv.cuh"

namespace er {

// Page scores of one (row, key head): the group's queries as int8 codes
// against the pages' int8 bounds, on the tensor cores. The dot products are
// exact integers (|I| <= 256 * 127^2 < 2^24, so float(I) is exact too) and the
// two roundings after them are in a fixed order: the scores, and so the
// choice, are the same on any grid.
//
// A warp takes 16 pages against 8 queries (m16n8k32): in each 64 channels a
// lane loads 16 consecutive codes of two pages, coalesced with its
// neighbours, and they serve as its share of two products' channels; the
// queries' codes lie in shared memory in the same order. (A lane a page, by
// dp4a, touches 32 lines a load: 35 us for 256 (row, key head) pairs of 512
// pages, and a page by 16 lanes with shuffles 47 us.)
constexpr int kScoreThreads = 512;

inline __host__ __device__ int codes_pitch(int d) { return (d + 63) / 64 * 64 + 16; }  // of a query's codes of one sign
inline __host__ __device__ int codes_bytes(int group, int d) {
  const int heads = (group + 7) / 8 * 8;
  return heads * 2 * codes_pitch(d) + heads * 4;
}

// The group's queries as codes, by the whole block: qc [heads][2][pitch], the
// negative ones, then the positive ones, zeros behind head_dim and the group;
// qt [heads], the steps. Returns whether a query is no number (no page ranks then).
template <typename TQ>
__device__ __forceinline__ bool code_queries(const TQ* q, int group, int d, int8_t* qc, float* qt) {
  const int lane = threadIdx.x & 31, heads = (group + 7) / 8 * 8, pitch = codes_pitch(d);
  bool none = false;
  for (int g = threadIdx.x >> 5; g < heads; g += blockDim.x >> 5) {
    float x[8], top = 0.f;  // head_dim is 256 at the most
    bool nan = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = lane + 32 * i;
      x[i] = g < group && c < d ? to_f32(q[(long long)g * d + c]) : 0.f;
      nan |= x[i] != x[i];
      top = fmaxf(top, fabsf(x[i]));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float t = top * kCodeStep;
    none |= __any_sync(0xffffffffu, nan) || !(t < INFINITY);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = lane + 32 * i;
      float r = t == 0.f ? 0.f : rintf(x[i] / t);
      r = r == r ? fminf(fmaxf(r, -127.f), 127.f) : 0.f;
      if (c < pitch) {
        qc[(g * 2 + 0) * pitch + c] = (int8_t)fminf(r, 0.f);
        qc[(g * 2 + 1) * pitch + c] = (int8_t)fmaxf(r, 0.f);
      }
    }
    if (lane == 0) qt[g] = t;
  }
  return __syncthreads_or(none);
}

__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 16 codes from channel c on, zeros behind head_dim (8-byte boundaries are all that is sure)
__device__ __forceinline__ uint4 load_codes(const int8_t* row, int c, int d) {
  uint4 x = make_uint4(0, 0, 0, 0);
  if (row && c < d) {
    if ((d & 15) == 0) {
      x = *reinterpret_cast<const uint4*>(row + c);
    } else {
      const uint2 lo = *reinterpret_cast<const uint2*>(row + c);
      x.x = lo.x;
      x.y = lo.y;
      if (c + 8 < d) {
        const uint2 hi = *reinterpret_cast<const uint2*>(row + c + 8);
        x.z = hi.x;
        x.w = hi.y;
      }
    }
  }
  return x;
}

// Scores of the pages [first, last) of a sequence; emit(o, score) by one lane each.
template <typename Emit>
__device__ __forceinline__ void score_pages(const KvView& kv, int seq, int h, int first, int last, int group,
                                            const int8_t* qc, const float* qt, bool none, const int8_t* codes,
                                            const float* scales, int* status, Emit emit) {
  const int d = kv.d, lane = threadIdx.x & 31, r = lane / 4, q = lane % 4, pitch = codes_pitch(d);
  const int32_t* table = kv.pages_of(seq);
  for (int o0 = first + (int)(threadIdx.x >> 5) * 16; o0 < last; o0 += (int)(blockDim.x >> 5) * 16) {
    const int8_t* row[2];
    float scale[2], best[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int o = o0 + r + 8 * i, page = o < last ? table[o] : -1;
      const bool ok = page >= 0 && page < kv.num_pages;
      if (o < last && !ok && q == 0) kv_report(status, ER_KV_BAD_PAGE);
      const long long at = ok ? (long long)page * kv.kv_heads + h : 0;
      row[i] = ok ? codes + at * 2 * d : nullptr;
      scale[i] = ok ? scales[at] : __int_as_float(0x7fc00000);
    }
#pragma unroll 1
    for (int g0 = 0; g0 < group; g0 += 8) {
      int sum[4] = {0, 0, 0, 0};
#pragma unroll 2
      for (int c0 = 0; c0 < d; c0 += 64) {
        const int c = c0 + q * 16;
        uint4 x[2][2];  // [least, greatest][page]
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          x[0][i] = load_codes(row[i], c, d);
          x[1][i] = load_codes(row[i] ? row[i] + d : nullptr, c, d);
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const uint4 b = *reinterpret_cast<const uint4*>(qc + ((g0 + r) * 2 + s) * pitch + c);
          mma_s8(sum, x[s][0].x, x[s][1].x, x[s][0].y, x[s][1].y, b.x, b.y);
          mma_s8(sum, x[s][0].z, x[s][1].z, x[s][0].w, x[s][1].w, b.z, b.w);
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {  // page r + 8 (e / 2), query 2 q + e % 2
        const int g = g0 + q * 2 + (e & 1);
        if (g < group) best[e >> 1] = fmaxf(best[e >> 1], __fmul_rn((float)sum[e], qt[g]));
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      best[i] = fmaxf(best[i], __shfl_xor_sync(0xffffffffu, best[i], 1));
      best[i] = fmaxf(best[i], __shfl_xor_sync(0xffffffffu, best[i], 2));
      const int o = o0 + r + 8 * i;
      if (q == 0 && o < last) emit(o, none ? __int_as_float(0x7fc00000) : __fmul_rn(best[i], scale[i]));
    }
  }
}

// What a row asks for: its sequence and how many pages that has, 0 when something is wrong with it.
__device__ __forceinline__ int row_pages(const KvView& kv, const int32_t* seqs, const int32_t* lens, int row, int* seq,
                                         int* bad) {
  *seq = seqs ? seqs[row] : row;
  const int len = lens[row];
  *bad = *seq < 0 || *seq >= kv.seqs ? ER_KV_BAD_SEQ : len < 0 || len > kv.capacity() ? ER_KV_BAD_LENGTH : 0;
  return *bad ? 0 : (int)(((long long)len + kv.page_size - 1) / kv.page_size);
}

// The rank keys of n scores into shared memory, four scores a load from the first 16-byte boundary on.
__device__ __forceinline__ void hold_keys(const float* scores, int n, uint32_t* held) {
  const int skip = min(n, (int)((16 - ((uintptr_t)scores & 15)) & 15) / 4), quads = (n - skip) / 4;
  if ((int)threadIdx.x < skip) held[HeldKeys::at(threadIdx.x)] = rank_key(scores[threadIdx.x]);
#pragma unroll 8
  for (int q = threadIdx.x; q < quads; q += blockDim.x) {
    const float4 x = *reinterpret_cast<const float4*>(scores + skip + q * 4);
    const int i = skip + q * 4;
    const uint4 k = make_uint4(rank_key(x.x), rank_key(x.y), rank_key(x.z), rank_key(x.w));
    if (skip == 0) {
      *reinterpret_cast<uint4*>(held + HeldKeys::at(i)) = k;
    } else {
      held[HeldKeys::at(i)] = k.x;
      held[HeldKeys::at(i + 1)] = k.y;
      held[HeldKeys::at(i + 2)] = k.z;
      held[HeldKeys::at(i + 3)] = k.w;
    }
  }
  const int i = skip + quads * 4 + threadIdx.x;
  if (i < n) held[HeldKeys::at(i)] = rank_key(scores[i]);
  __syncthreads();
}

constexpr size_t kSelectSmem = 220 * 1024;  // of a CTA that chooses: histograms, codes, keys

// Positions that rank r of a cluster holds: `each` of them, a multiple of 4.
__host__ __device__ inline int cluster_each(int n) { return (n + 4 * kClusterCtas - 1) / (4 * kClusterCtas) * 4; }

// How a (sequence, key head)'s positions are chosen from: by a CTA alone; or
// by a cluster, whose first CTA chooses, or whose CTAs choose together.
enum ChooseMode { kAlone, kFirst, kTogether };
// Few units run as clusters, all at once, and those choose together where
// there is much to choose from: every pass of the choice then reads the
// histograms of 8 CTAs, which small ones do not repay. (Eviction to 512 of
// 16 units, by the first CTA and together: of 2048 positions 13.8 and 29.6 us,
// 4096 16.7 and 29.9, 8192 21.7 and 31.1, 12288 36.5 and 28.3, 16384 41.3 and
// 29.1, 32768 61.6 and 32.5; 64 pages of one position each, 4 queries a key head:
// 8192 23.2 and 31.9, 16384 36.3 and 39.7, 32768 71.6 and 56.4. With 4 and 32
// units eviction crosses at the same place.) Otherwise a CTA a unit, unless
// its shared memory cannot hold the keys beside `beside` bytes.
inline int choose_mode(long long units, int n, size_t beside) {
  if (select_bytes(n) + held_bytes(n) + beside > kSelectSmem) return kTogether;
  return units * kClusterCtas > 148 * 2 ? kAlone : n > 8192 ? kTogether : kFirst;
}
inline int choose_held(int mode, int n) { return mode == kTogether ? cluster_each(n) : n; }  // keys a CTA holds

// Scores and choice of one (row, key head); in a cluster each CTA scores an
// eighth of the pages.
template <typename TQ, int MODE>
__global__ void __launch_bounds__(kScoreThreads)
    kv_pick_kernel(KvView kv, const TQ* __restrict__ q, long long q_stride, int group, const int32_t* __restrict__ seqs,
                   const int32_t* __restrict__ lens, const int8_t* __restrict__ codes,
                   const float* __restrict__ scales, int most, int budget, int sinks, int recent,
                   int32_t* __restrict__ pages, int32_t* __restrict__ counts, int* status) {
  constexpr bool CLUSTER = MODE != kAlone;
  extern __shared__ __align__(16) char sm[];
  __shared__ SelectScratch sc;
  int* hist = reinterpret_cast<int*>(sm);
  int8_t* qc = reinterpret_cast<int8_t*>(sm + select_bytes(most));
  float* qt = reinterpret_cast<float*>(qc + (group + 7) / 8 * 16 * codes_pitch(kv.d));
  uint32_t* held = reinterpret_cast<uint32_t*>(qc + codes_bytes(group, kv.d));
  kv_enter();
  const int unit = CLUSTER ? blockIdx.x / kClusterCtas : blockIdx.x, rank = CLUSTER ? cluster_rank() : 0;
  const int row = unit / kv.kv_heads, h = unit % kv.kv_heads;
  int seq, bad;
  const int np = row_pages(kv, seqs, lens, row, &seq, &bad);
  if (bad && rank == 0 && threadIdx.x == 0) kv_report(status, bad);
  int32_t* out = pages + (long long)unit * budget;
  const int take = min(np, budget);
  if (np > budget) {
    const bool none =
        code_queries(q + (long long)row * q_stride + (long long)h * group * kv.d, group, kv.d, qc, qt);
    if (MODE == kFirst) cluster_sync();  // the first CTA runs: its shared memory can be written
    const int each = CLUSTER ? cluster_each(np) : np;
    const int first = min(np, rank * each), last = min(np, first + each);
    const uint32_t to = MODE == kFirst ? cluster_addr(smem_addr(held), 0) : 0;
    score_pages(kv, seq, h, first, last, group, qc, qt, none, codes, scales, status, [&](int o, float v) {
      if (MODE == kFirst)
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to + HeldKeys::at(o) * 4), "r"(rank_key(v)) : "memory");
      else
        held[HeldKeys::at(o - first)] = rank_key(v);
    });
    if (MODE == kFirst)
      cluster_sync();
    else
      __syncthreads();
    const int b0 = MODE == kTogether ? first : 0, nl = MODE == kTogether ? last - first : np;
    if (MODE == kTogether || rank == 0)
      take_best<MODE == kTogether ? kClusterCtas : 1>(HeldKeys{held}, b0, nl, np, budget, sinks, recent, hist, sc,
                                                      [&](int slot, int i) { out[slot] = i; });
  } else if (rank == 0) {  // all are taken, whatever they score
    for (int i = threadIdx.x; i < budget; i += kScoreThreads) out[i] = i < np ? i : -1;
  }
  if (rank == 0 && threadIdx.x == 0) counts[unit] = take;
}

struct MassView {
  const float* mass;
  float* to_mass;
  long long seq_stride, head_stride, to_seq_stride, to_head_stride;
  int len, to_len;
};

// Copies a (sequence, key head)'s kept rows into the destination's pages, by
// warps `warp`, warp + warps, .. : the lanes split a row's 16-byte columns,
// lane groups the rows, four rows of a lane under way at once (list, pages
// and values are three waits, one after the other).
__device__ __forceinline__ void move_rows(const KvView& from, const KvView& to, int seq, int h, const int32_t* list,
                                          int n, int row_bytes, int warp, int warps, int* status) {
  constexpr int N = 4;
  const int cols = row_bytes / 16, lane = threadIdx.x & 31;  // 1 .. 64 columns
  int wide = 1;
  while (wide < cols && wide < 32) wide *= 2;
  const int per = 32 / wide, col = lane % wide;
  const int32_t *ft = from.pages_of(seq), *tt = to.pages_of(seq);
#pragma unroll 1
  for (int s0 = warp * per * N + lane / wide; s0 < n; s0 += warps * per * N) {
    int src[N], pa[N], pb[N];
#pragma unroll
    for (int j = 0; j < N; ++j) src[j] = s0 + j * per < n ? list[s0 + j * per] : -1;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      pa[j] = src[j] >= 0 ? ft[from.ordinal(src[j])] : 0;
      pb[j] = src[j] >= 0 ? tt[to.ordinal(s0 + j * per)] : 0;
    }
#pragma unroll 1
    for (int c = col; c < cols; c += 32) {
      uint4 x[N], y[N];
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if (src[j] < 0) continue;
        if (pa[j] < 0 || pa[j] >= from.num_pages || pb[j] < 0 || pb[j] >= to.num_pages) {
          if (c == 0) kv_report(status, ER_KV_BAD_PAGE);
          src[j] = -1;
          continue;
        }
        const long long so =
            pa[j] * from.page_stride + h * from.head_stride + from.slot(src[j]) * from.slot_stride + c * 16;
        x[j] = ld_stream_u4(from.k + so);
        y[j] = ld_stream_u4(from.v + so);
      }
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if (src[j] < 0) continue;
        const long long de =
            pb[j] * to.page_stride + h * to.head_stride + to.slot(s0 + j * per) * to.slot_stride + c * 16;
        *reinterpret_cast<uint4*>(to.k + de) = x[j];
        *reinterpret_cast<uint4*>(to.v + de) = y[j];
      }
    }
  }
}

// The kept positions of a (sequence, key head) and their weights. A cluster
// moves the rows, too; for CTAs alone kv_move_kernel does.
template <int MODE>
__global__ void __launch_bounds__(1024)
    kv_keep_kernel(KvView kv, KvView dst, MassView m, const int32_t* __restrict__ lens, int most, int budget, int sinks,
                   int recent, int row_bytes, int32_t* kept, int32_t* __restrict__ lens_out, int* status) {
  constexpr bool CLUSTER = MODE != kAlone;
  extern __shared__ __align__(16) char sm[];
  __shared__ SelectScratch sc;
  int* hist = reinterpret_cast<int*>(sm);
  uint32_t* held = reinterpret_cast<uint32_t*>(sm + select_bytes(most));
  kv_enter();
  const int unit = CLUSTER ? blockIdx.x / kClusterCtas : blockIdx.x, rank = CLUSTER ? cluster_rank() : 0;
  const int seq = unit / kv.kv_heads, h = unit % kv.kv_heads;
  int n = lens[seq];
  if (n < 0 || n > kv.capacity() || n > m.len) {
    if (threadIdx.x == 0 && h == 0 && rank == 0) kv_report(status, ER_KV_BAD_LENGTH);
    n = 0;
  }
  const float* w = m.mass + seq * m.seq_stride + h * m.head_stride;
  int32_t* out = kept + (long long)unit * budget;
  const int take = min(n, budget), ctas = CLUSTER ? kClusterCtas : 1;
  const int t0 = rank * blockDim.x + threadIdx.x, threads = ctas * blockDim.x;
  if (n > budget) {
    if (MODE == kTogether || rank == 0) {
      const int each = MODE == kTogether ? cluster_each(n) : n, first = min(n, rank * each), last = min(n, first + each);
      hold_keys(w + first, last - first, held);
      take_best<MODE == kTogether ? kClusterCtas : 1>(HeldKeys{held}, first, last - first, n, budget, sinks, recent, hist,
                                                      sc, [&](int slot, int i) { out[slot] = i; });
    }
  } else {
    for (int i = t0; i < budget; i += threads) out[i] = i < n ? i : -1;
  }
  if (CLUSTER)
    cluster_sync();
  else
    __syncthreads();  // the list is written
  if (t0 == 0 && h == 0) lens_out[seq] = take;
  float* to = m.to_mass + seq * m.to_seq_stride + h * m.to_head_stride;
#pragma unroll 4
  for (int i = t0; i < take; i += threads) to[i] = w[out[i]];
  if (CLUSTER)
    move_rows(kv, dst, seq, h, out, take, row_bytes, rank * (blockDim.x >> 5) + (threadIdx.x >> 5),
              kClusterCtas * (blockDim.x >> 5), status);
}

// The rows of the kept positions. At 16 sequences of 8 key heads cut to 4096
// positions of 256 + 256 bytes it moves 6.3 TB/s.
__global__ void __launch_bounds__(256) kv_move_kernel(KvView from, KvView to, const int32_t* __restrict__ kept,
                                                      int budget, int row_bytes, int* status) {
  kv_enter();
  move_rows(from, to, blockIdx.y, blockIdx.z, kept + ((long long)blockIdx.y * from.kv_heads + blockIdx.z) * budget,
            budget, row_bytes, blockIdx.x * 8 + (threadIdx.x >> 5), gridDim.x * 8, status);
}

}  // namespace er

using namespace er;

namespace {

size_t pick_smem(int most, int group, int d) { return select_bytes(most) + codes_bytes(group, d) + held_bytes(most); }

template <typename TQ>
int pick_go(const KvView& kv, const void* q, long long q_stride, int units, int group, const int32_t* seqs,
            const int32_t* lens, const int8_t* codes, const float* scales, int budget, int sinks, int recent,
            int32_t* pages, int32_t* counts, int* status, cudaStream_t st) {
  const int mode = choose_mode(units, kv.width, codes_bytes(group, kv.d)), most = choose_held(mode, kv.width);
  auto kernel = mode == kTogether ? kv_pick_kernel<TQ, kTogether>
                : mode == kFirst  ? kv_pick_kernel<TQ, kFirst>
                                  : kv_pick_kernel<TQ, kAlone>;
  static std::atomic<unsigned long long> done[3];
  if (int rc = allow_smem(kernel, kSelectSmem, done[mode])) return rc;
  const bool cluster = mode != kAlone;
  return kv_launch(kernel, dim3(cluster ? units * kClusterCtas : units), kScoreThreads, pick_smem(most, group, kv.d),
                   cluster, st, "kv_pick_kernel", kv, (const TQ*)q, q_stride, group, seqs, lens, codes, scales, most,
                   budget, sinks, recent, pages, counts, status);
}

}  // namespace

extern "C" int er_kv_select(const er_kv_cache* cache, const void* q, int q_dtype, long long q_stride, int rows,
                            int heads, const int32_t* seqs, const int32_t* lens, const int8_t* codes,
                            const float* scales, int budget, int sinks, int recent, int32_t* pages_out,
                            int32_t* counts_out, int* status, void* stream) {
  if (int rc = kv_check("er_kv_select", cache)) return rc;
  if (rows < 0 || heads <= 0 || heads > kMaxHeads || heads % cache->kv_heads)
    return fail(ER_EINVAL, "er_kv_select: rows %d, heads %d / %d", rows, heads, cache->kv_heads);
  if (q_dtype != ER_DTYPE_F32 && q_dtype != ER_DTYPE_BF16) return fail(ER_EINVAL, "er_kv_select: q dtype %d", q_dtype);
  if (budget <= 0 || sinks < 0 || recent < 0 || (long long)sinks + recent > budget)
    return fail(ER_EINVAL, "er_kv_select: budget %d with %d first and %d last pages", budget, sinks, recent);
  if (q_stride < (long long)heads * cache->head_dim)
    return fail(ER_EINVAL, "er_kv_select: row stride %lld shorter than the queries", q_stride);
  if (!seqs && rows > cache->seqs) return fail(ER_EINVAL, "er_kv_select: %d rows, %d sequences", rows, cache->seqs);
  if (rows == 0) return ER_OK;
  if (!q || !lens || !codes || !scales || !pages_out || !counts_out) return fail(ER_EINVAL, "er_kv_select: null pointer");
  if (((uintptr_t)codes & 15)) return fail(ER_EINVAL, "er_kv_select: codes must be 16-byte aligned");
  const int group = heads / cache->kv_heads;
  if (group > 64) return fail(ER_EINVAL, "er_kv_select: %d queries a key head (at most 64)", group);
  if ((long long)rows * cache->kv_heads > 0x7fffffff / kClusterCtas)
    return fail(ER_EINVAL, "er_kv_select: %d rows of %d key heads", rows, cache->kv_heads);
  if (pick_smem(cluster_each(cache->table_width), group, cache->head_dim) > kSelectSmem)
    return fail(ER_EINVAL, "er_kv_select: a table of %d pages (about 300000 fit)", cache->table_width);
  const KvView kv = kv_view(*cache);
  const int units = rows * kv.kv_heads;
  return q_dtype == ER_DTYPE_BF16
             ? pick_go<__nv_bfloat16>(kv, q, q_stride, units, group, seqs, lens, codes, scales, budget, sinks, recent,
                                      pages_out, counts_out, status, (cudaStream_t)stream)
             : pick_go<float>(kv, q, q_stride, units, group, seqs, lens, codes, scales, budget, sinks, recent, pages_out,
                              counts_out, status, (cudaStream_t)stream);
}

extern "C" int er_kv_evict(const er_kv_cache* from, const er_kv_cache* to, const int32_t* lens, const float* mass,
                           long long mass_seq_stride, long long mass_head_stride, int mass_len, float* to_mass,
                           long long to_mass_seq_stride, long long to_mass_head_stride, int to_mass_len, int budget,
                           int sinks, int recent, int32_t* kept_out, int32_t* lens_out, int* status, void* stream) {
  if (int rc = kv_check("er_kv_evict", from)) return rc;
  if (int rc = kv_check("er_kv_evict", to)) return rc;
  if (from->dtype != to->dtype || from->kv_heads != to->kv_heads || from->head_dim != to->head_dim ||
      from->seqs != to->seqs)
    return fail(ER_EINVAL, "er_kv_evict: the two caches differ in type, key heads, head_dim or sequences");
  if (budget <= 0 || sinks < 0 || recent < 0 || (long long)sinks + recent > budget)
    return fail(ER_EINVAL, "er_kv_evict: budget %d with %d first and %d last positions", budget, sinks, recent);
  if (mass_len < 0 || to_mass_len < budget || (long long)to->table_width * to->page_size < budget)
    return fail(ER_EINVAL, "er_kv_evict: budget %d, but the destination holds %lld positions and %d weights", budget,
                (long long)to->table_width * to->page_size, to_mass_len);
  if (from->seqs == 0) return ER_OK;
  if (!lens || !mass || !to_mass || !kept_out || !lens_out) return fail(ER_EINVAL, "er_kv_evict: null pointer");
  if (lens == lens_out) return fail(ER_EINVAL, "er_kv_evict: lens_out is lens");
  if (from->seqs > 65535) return fail(ER_EINVAL, "er_kv_evict: %d sequences (at most 65535)", from->seqs);
  const KvView a = kv_view(*from), b = kv_view(*to);
  const MassView m{mass,        to_mass,  mass_seq_stride, mass_head_stride, to_mass_seq_stride, to_mass_head_stride,
                   mass_len, to_mass_len};
  cudaStream_t st = (cudaStream_t)stream;
  const int row_bytes = a.d * (from->dtype == ER_DTYPE_BF16 ? 2 : 4), units = a.seqs * a.kv_heads;
  if (select_bytes(cluster_each(mass_len)) + held_bytes(cluster_each(mass_len)) > kSelectSmem)
    return fail(ER_EINVAL, "er_kv_evict: %d weights a key head (about 370000 fit)", mass_len);
  const int mode = choose_mode(units, mass_len, 0), most = choose_held(mode, mass_len);
  auto keep = mode == kTogether ? kv_keep_kernel<kTogether>
              : mode == kFirst ? kv_keep_kernel<kFirst>
                                   : kv_keep_kernel<kAlone>;
  static std::atomic<unsigned long long> done[3];
  if (int rc = allow_smem(keep, kSelectSmem, done[mode])) return rc;
  const bool cluster = mode != kAlone;
  if (int rc = kv_launch(keep, dim3(cluster ? units * kClusterCtas : units),
                         most <= 1024 ? 256 : most <= 8192 ? 512 : 1024, select_bytes(most) + held_bytes(most), cluster,
                         st, "kv_keep_kernel", a, b, m, lens, most, budget, sinks, recent, row_bytes, kept_out, lens_out,
                         status))
    return rc;
  if (cluster) return ER_OK;
  const long long want = 148 * 32 / ((long long)a.seqs * a.kv_heads) + 1;
  const long long first_rows = (budget + 31) / 32;  // rows of a warp's first round, times 8
  const dim3 grid((unsigned)(first_rows < want ? first_rows : want), a.seqs, a.kv_heads);
  return launch_chained(kv_move_kernel, grid, dim3(256), 0, st, "kv_move_kernel", a, b, (const int32_t*)kept_out,
                        budget, row_bytes, status);
}
