// er_kv_select.cu -- the pages worth reading for each query, and the
// positions worth keeping in a cache that grows too long.
//
// Both rank by a score and take the best: a radix select by the whole CTA
// (er_kv.cuh) finds the score of the last one taken, a second pass in
// position order writes the taken ones ascending, equal scores to the lower
// position.
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

// Scores alone, for tables too wide for shared memory.
template <typename TQ>
__global__ void __launch_bounds__(kScoreThreads)
    kv_score_kernel(KvView kv, const TQ* __restrict__ q, long long q_stride, int group, const int32_t* __restrict__ seqs,
                    const int32_t* __restrict__ lens, const int8_t* __restrict__ codes,
                    const float* __restrict__ scales, float* __restrict__ scores, int* status) {
  extern __shared__ __align__(16) int8_t qc[];
  float* qt = reinterpret_cast<float*>(qc + (group + 7) / 8 * 16 * codes_pitch(kv.d));
  kv_enter();
  const int row = blockIdx.y / kv.kv_heads, h = blockIdx.y % kv.kv_heads;
  int seq, bad;
  const int np = row_pages(kv, seqs, lens, row, &seq, &bad);  // what is wrong is reported by the choice
  if (np == 0) return;
  const bool none = code_queries(q + (long long)row * q_stride + (long long)h * group * kv.d, group, kv.d, qc, qt);
  float* out = scores + (long long)blockIdx.y * kv.width;
  const int each = (np + gridDim.x - 1) / gridDim.x, first = min(np, (int)blockIdx.x * each);
  score_pages(kv, seq, h, first, min(np, first + each), group, qc, qt, none, codes, scales, status,
              [&](int o, float v) { out[o] = v; });
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

// Writes, ascending, the `take` of n positions that are forced (the first
// `sinks`, the last `recent`) or rank best; emit(slot, i) for each.
template <typename Keys, typename Emit>
__device__ __forceinline__ void take_best(const Keys& keys, int n, int take, int sinks, int recent, int* hist, int* red,
                                          Emit emit) {
  if (n <= take) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) emit(i, i);
    return;
  }
  const int lo = sinks, hi = n - recent, want = take - sinks - recent;
  uint32_t least = 0xffffffffu;
  int equal = 0;
  if (want > 0) least = block_select(keys, n, lo, hi, want, hist, red, &equal);
  // in rounds of a run of 4, 8, .. 32 positions a thread
  int run = 4;
  while (run < 32 && run * (int)blockDim.x < n) run *= 2;
  int above = 0, same = 0;  // taken outright, and equal to the threshold, so far
  for (int i0 = 0; i0 < n; i0 += run * blockDim.x) {
    const int b = i0 + (int)threadIdx.x * run;
    uint32_t sure = 0, tied = 0;  // of the run's positions
    for (int j = 0; j < run && b + j < n; j += 4) {
      const uint4 k4 = keys.four(b + j, n);
      const uint32_t k[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = b + j + e;
        const bool forced = i < lo || i >= hi;
        if (i < n) {
          sure |= (uint32_t)(forced || (want > 0 && k[e] > least)) << (j + e);
          tied |= (uint32_t)(!forced && want > 0 && k[e] == least) << (j + e);
        }
      }
    }
    // 16 bits each: a round has at most 32 * 1024 positions
    int all;
    const int before = block_scan(__popc(sure) | __popc(tied) << 16, red, &all);
    int at = above + (before & 0xffff), tie = same + (before >> 16);
    for (uint32_t left = sure | tied; left; left &= left - 1) {
      const int j = __ffs(left) - 1;
      if ((sure >> j) & 1) {
        emit(at + min(tie, equal), b + j);
        ++at;
      } else {
        if (tie < equal) emit(at + tie, b + j);
        ++tie;
      }
    }
    above += all & 0xffff;
    same += all >> 16;
  }
}

constexpr int kTakeThreads = 1024;

// Shared memory of a CTA that takes the best of at most n: the histograms,
// and the keys where they fit beside them (*held).
inline size_t take_smem(long long n, bool* held) {
  *held = select_bytes(n) + held_bytes(n) <= 200 * 1024;
  return select_bytes(n) + (*held ? held_bytes(n) : 0);
}
inline int take_threads(long long n) { return n <= 1024 ? 256 : n <= 8192 ? 512 : kTakeThreads; }

template <int THREADS, typename Keys>
__device__ __forceinline__ void write_choice(const Keys& keys, int n, int budget, int sinks, int recent, int* hist,
                                             int* red, int32_t* out, int32_t* count) {
  take_best(keys, n, budget, sinks, recent, hist, red, [&](int slot, int i) { out[slot] = i; });
  const int take = min(n, budget);
  for (int i = take + threadIdx.x; i < budget; i += THREADS) out[i] = -1;
  if (threadIdx.x == 0) *count = take;
}

// Scores and choice of one (row, key head) in one launch: a CTA, or with few
// units a cluster whose CTAs score an eighth of the pages each, straight into
// the shared memory of the first, which chooses.
template <typename TQ, bool CLUSTER>
__global__ void __launch_bounds__(kScoreThreads)
    kv_pick_kernel(KvView kv, const TQ* __restrict__ q, long long q_stride, int group, const int32_t* __restrict__ seqs,
                   const int32_t* __restrict__ lens, const int8_t* __restrict__ codes,
                   const float* __restrict__ scales, int budget, int sinks, int recent, int32_t* __restrict__ pages,
                   int32_t* __restrict__ counts, int* status) {
  extern __shared__ __align__(16) char sm[];
  __shared__ int red[kScoreThreads / 32 + 4];
  int* hist = reinterpret_cast<int*>(sm);
  int8_t* qc = reinterpret_cast<int8_t*>(sm + select_bytes(kv.width));
  float* qt = reinterpret_cast<float*>(qc + (group + 7) / 8 * 16 * codes_pitch(kv.d));
  uint32_t* held = reinterpret_cast<uint32_t*>(qc + codes_bytes(group, kv.d));
  kv_enter();
  const int unit = CLUSTER ? blockIdx.x / kClusterCtas : blockIdx.x, rank = CLUSTER ? cluster_rank() : 0;
  const int row = unit / kv.kv_heads, h = unit % kv.kv_heads;
  int seq, bad;
  const int np = row_pages(kv, seqs, lens, row, &seq, &bad);
  if (bad && rank == 0 && threadIdx.x == 0) kv_report(status, bad);
  if (np > budget) {  // else all are taken, whatever they score
    const bool none =
        code_queries(q + (long long)row * q_stride + (long long)h * group * kv.d, group, kv.d, qc, qt);
    if (CLUSTER) cluster_sync();  // the first CTA runs: its shared memory can be written
    const int first = CLUSTER ? (int)((long long)np * rank / kClusterCtas) : 0;
    const int last = CLUSTER ? (int)((long long)np * (rank + 1) / kClusterCtas) : np;
    const uint32_t to = CLUSTER ? cluster_addr(smem_addr(held), 0) : smem_addr(held);
    score_pages(kv, seq, h, first, last, group, qc, qt, none, codes, scales, status, [&](int o, float v) {
      const uint32_t at = to + HeldKeys::at(o) * 4, k = rank_key(v);
      if (CLUSTER)
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(k) : "memory");
      else
        asm volatile("st.shared.u32 [%0], %1;" ::"r"(at), "r"(k) : "memory");
    });
    if (CLUSTER)
      cluster_sync();
    else
      __syncthreads();
  }
  if (rank == 0)
    write_choice<kScoreThreads>(HeldKeys{held}, np, budget, sinks, recent, hist, red,
                                pages + (long long)unit * budget, counts + unit);
}

// The choice alone, from scores in memory.
__global__ void __launch_bounds__(kTakeThreads)
    kv_choose_kernel(KvView kv, const int32_t* __restrict__ seqs, const int32_t* __restrict__ lens,
                     const float* __restrict__ scores, int budget, int sinks, int recent,
                     int32_t* __restrict__ pages, int32_t* __restrict__ counts, int* status) {
  extern __shared__ int hist[];
  __shared__ int red[kTakeThreads / 32 + 4];
  kv_enter();
  int seq, bad;
  const int n = row_pages(kv, seqs, lens, blockIdx.x / kv.kv_heads, &seq, &bad);
  if (bad && threadIdx.x == 0) kv_report(status, bad);
  write_choice<kTakeThreads>(ScoreKeys{scores + (long long)blockIdx.x * kv.width}, n, budget, sinks, recent, hist, red,
                             pages + (long long)blockIdx.x * budget, counts + blockIdx.x);
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

// The kept positions of a (sequence, key head) and their weights, by a CTA.
// CLUSTER (few units): by the first CTA of a cluster, whose CTAs then move the
// rows together; otherwise kv_move_kernel moves them.
template <bool CLUSTER>
__global__ void __launch_bounds__(kTakeThreads)
    kv_keep_kernel(KvView kv, KvView dst, MassView m, const int32_t* __restrict__ lens, int budget, int sinks,
                   int recent, int held, int row_bytes, int32_t* kept, int32_t* __restrict__ lens_out, int* status) {
  extern __shared__ int hist[];
  __shared__ int red[kTakeThreads / 32 + 4];
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
  const int take = min(n, budget);
  if (rank == 0) {
    auto emit = [&](int slot, int i) { out[slot] = i; };
    if (held) {
      uint32_t* keys = (uint32_t*)(hist + select_bytes(m.len) / 4);
      if (n > budget) hold_keys(w, n, keys);
      take_best(HeldKeys{keys}, n, budget, sinks, recent, hist, red, emit);
    } else {
      take_best(ScoreKeys{w}, n, budget, sinks, recent, hist, red, emit);
    }
    for (int i = take + threadIdx.x; i < budget; i += blockDim.x) out[i] = -1;
    if (threadIdx.x == 0 && h == 0) lens_out[seq] = take;
  }
  if (CLUSTER)
    cluster_sync();  // the list is written
  else
    __syncthreads();
  if (rank == 0) {
    float* to = m.to_mass + seq * m.to_seq_stride + h * m.to_head_stride;
#pragma unroll 4
    for (int i = threadIdx.x; i < take; i += blockDim.x) to[i] = w[out[i]];
  }
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

// Shared memory of kv_pick_kernel; more than kPickSmem means that the scores go through the workspace.
constexpr size_t kPickSmem = 200 * 1024;
size_t pick_smem(int width, int group, int d) { return select_bytes(width) + codes_bytes(group, d) + held_bytes(width); }

template <typename TQ>
int pick_go(const KvView& kv, const void* q, long long q_stride, int units, int group, const int32_t* seqs,
            const int32_t* lens, const int8_t* codes, const float* scales, int budget, int sinks, int recent,
            int32_t* pages, int32_t* counts, int* status, cudaStream_t st) {
  const size_t smem = pick_smem(kv.width, group, kv.d);
  const bool cluster = units * kClusterCtas <= 148 * 2;  // all at once
  auto kernel = cluster ? kv_pick_kernel<TQ, true> : kv_pick_kernel<TQ, false>;
  static std::atomic<unsigned long long> done[2];
  if (int rc = allow_smem(kernel, kPickSmem, done[cluster])) return rc;
  return kv_launch(kernel, dim3(cluster ? units * kClusterCtas : units), kScoreThreads, smem, cluster, st,
                   "kv_pick_kernel", kv, (const TQ*)q, q_stride, group, seqs, lens, codes, scales, budget, sinks,
                   recent, pages, counts, status);
}

}  // namespace

extern "C" size_t er_kv_select_workspace_bytes(const er_kv_cache* cache, int rows, int heads) {
  if (!cache || rows <= 0 || cache->kv_heads <= 0 || heads <= 0 || cache->table_width <= 0) return 0;
  if (pick_smem(cache->table_width, heads / cache->kv_heads, cache->head_dim) <= kPickSmem) return 0;
  return align_up((size_t)rows * cache->kv_heads * cache->table_width * sizeof(float), 256);
}

extern "C" int er_kv_select(const er_kv_cache* cache, const void* q, int q_dtype, long long q_stride, int rows,
                            int heads, const int32_t* seqs, const int32_t* lens, const int8_t* codes,
                            const float* scales, int budget, int sinks, int recent, int32_t* pages_out,
                            int32_t* counts_out, int* status, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = kv_check("er_kv_select", cache)) return rc;
  if (rows < 0 || heads <= 0 || heads % cache->kv_heads)
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
  const size_t smem = codes_bytes(group, cache->head_dim);
  if (smem > 40 * 1024) return fail(ER_EINVAL, "er_kv_select: %d queries a key head", group);
  if ((long long)rows * cache->kv_heads > 65535)
    return fail(ER_EINVAL, "er_kv_select: %d rows of %d key heads (at most 65535 in all)", rows, cache->kv_heads);
  const size_t need = er_kv_select_workspace_bytes(cache, rows, heads);
  if (need && (!workspace || workspace_bytes < need))
    return fail(ER_ENOSPACE, "er_kv_select: workspace %zu bytes, need %zu", workspace_bytes, need);
  const KvView kv = kv_view(*cache);
  cudaStream_t st = (cudaStream_t)stream;
  const int units = rows * kv.kv_heads;
  const bool qb = q_dtype == ER_DTYPE_BF16;
  if (!need)
    return qb ? pick_go<__nv_bfloat16>(kv, q, q_stride, units, group, seqs, lens, codes, scales, budget, sinks, recent,
                                       pages_out, counts_out, status, st)
              : pick_go<float>(kv, q, q_stride, units, group, seqs, lens, codes, scales, budget, sinks, recent,
                               pages_out, counts_out, status, st);
  const dim3 grid((unsigned)(148 * 4 / units + 1), units);
  float* scores = (float*)workspace;
  int rc = qb ? launch_chained(kv_score_kernel<__nv_bfloat16>, grid, dim3(kScoreThreads), smem, st, "kv_score_kernel",
                               kv, (const __nv_bfloat16*)q, q_stride, group, seqs, lens, codes, scales, scores, status)
              : launch_chained(kv_score_kernel<float>, grid, dim3(kScoreThreads), smem, st, "kv_score_kernel", kv,
                               (const float*)q, q_stride, group, seqs, lens, codes, scales, scores, status);
  if (rc) return rc;
  return launch_chained(kv_choose_kernel, dim3(units), dim3(kTakeThreads), select_bytes(kv.width), st, "kv_choose_kernel", kv,
                        seqs, lens, (const float*)scores, budget, sinks, recent, pages_out, counts_out, status);
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
  if (from->seqs > 65535 || from->kv_heads > 65535)
    return fail(ER_EINVAL, "er_kv_evict: %d sequences, %d key heads", from->seqs, from->kv_heads);
  const KvView a = kv_view(*from), b = kv_view(*to);
  const MassView m{mass,        to_mass,  mass_seq_stride, mass_head_stride, to_mass_seq_stride, to_mass_head_stride,
                   mass_len, to_mass_len};
  cudaStream_t st = (cudaStream_t)stream;
  bool held;
  const size_t take = take_smem(mass_len, &held);
  const int row_bytes = a.d * (from->dtype == ER_DTYPE_BF16 ? 2 : 4), units = a.seqs * a.kv_heads;
  // clusters all at once, each with little to move beside the choice (the
  // second launch costs about what 64 MB take to move)
  const bool cluster = units * kClusterCtas <= 148 * 2 && 2LL * units * budget * row_bytes <= 64ll << 20;
  static std::atomic<unsigned long long> done[2];
  if (int rc = cluster ? allow_smem(kv_keep_kernel<true>, 200 * 1024, done[1])
                       : allow_smem(kv_keep_kernel<false>, 200 * 1024, done[0]))
    return rc;
  if (int rc = kv_launch(cluster ? kv_keep_kernel<true> : kv_keep_kernel<false>,
                         dim3(cluster ? units * kClusterCtas : units), take_threads(mass_len), take, cluster, st,
                         "kv_keep_kernel", a, b, m, lens, budget, sinks, recent, (int)held, row_bytes, kept_out,
                         lens_out, status))
    return rc;
  if (cluster) return ER_OK;
  const long long want = 148 * 32 / ((long long)a.seqs * a.kv_heads) + 1;
  const long long most = (budget + 31) / 32;  // rows of a warp's first round, times 8
  const dim3 grid((unsigned)(most < want ? most : want), a.seqs, a.kv_heads);
  return launch_chained(kv_move_kernel, grid, dim3(256), 0, st, "kv_move_kernel", a, b, (const int32_t*)kept_out,
                        budget, row_bytes, status);
}
