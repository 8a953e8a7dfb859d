// er_beam.cu -- beam search's choice of continuations: of every batch's
// beams x vocabulary candidates of value score + log softmax(logits)[token]
// the best `count`.
//
// The logits are read once. Within a beam the value rises with the logit, so a
// CTA that reads a part of a row keeps the part's best `count` logits (the
// other candidates cannot be chosen) beside the part's maximum and sum of
// exponentials; a second kernel joins the parts' sums and chooses among what
// was kept, by values in 64 bits: candidates of different beams compare through
// their beams' log-sums, whose rounding in 32 bits would decide close ones.
// 4 bytes a candidate and about a dozen instructions: memory bounds it.
#include "er_kv.cuh"

namespace er {

namespace {

constexpr int kScanThreads = 256, kEach = 16, kTile = kScanThreads * kEach;  // logits a tile
constexpr int kMaxCount = 128, kMaxBeams = 1024;
constexpr int kHeld = kTile + kMaxCount;  // what a CTA may hold before it has to choose

struct BeamArgs {
  const void* logits;
  long long stride;
  const float* scores;
  int batch, beams, vocab, count;
  int parts, part;  // of a row, and logits of each (a multiple of the tile)
  double* sums;     // [rows][parts] of 2^.. relative to maxima
  float* maxima;    // [rows][parts]
  unsigned long long* kept;  // [rows][parts][count]: rank key of the logit, then ~token; 0 behind the last
  float* scores_out;
  int32_t *beams_out, *tokens_out;
};

// keys that rank as the pair (logit, lower token first)
__device__ __forceinline__ unsigned long long pack(float x, int token) {
  return (unsigned long long)rank_key(x) << 32 | (uint32_t)~token;
}
__device__ __forceinline__ float unrank(uint32_t k) {
  return k & 0x80000000u ? __uint_as_float(k & 0x7fffffffu) : __uint_as_float(~k);
}

// Sum of a count over the block, the same in all threads; `red`: two words a warp, used in turn.
struct BlockCount {
  int* red;
  int turn;
  __device__ __forceinline__ int operator()(int v) {
    int* r = red + turn * 32;
    turn ^= 1;
    v = __reduce_add_sync(0xffffffffu, v);
    if ((threadIdx.x & 31) == 0) r[threadIdx.x >> 5] = v;
    __syncthreads();
    const int lane = threadIdx.x & 31;
    return __reduce_add_sync(0xffffffffu, lane < (int)(blockDim.x >> 5) ? r[lane] : 0);
  }
};

// A bound that exactly `want` of the block's distinct keys reach (has(t): how
// many of the thread's keys are >= t), by halving; `least` .. `most`: such that
// all, or more than `want`, reach the one and less than `want` the other + 1.
template <typename Has>
__device__ __forceinline__ unsigned long long bound_of(int want, unsigned long long least, unsigned long long most,
                                                       BlockCount& count, Has has) {
  while (least < most) {
    const unsigned long long mid = least + (most - least) / 2 + 1;
    const int n = count(has(mid));
    if (n == want) return mid;
    if (n > want)
      least = mid;
    else
      most = mid - 1;
  }
  return least;
}

template <typename T>
__device__ __forceinline__ void load_tile(const T* row, int i0, int end, bool wide, float (&x)[kEach]) {
  // thread t has logits 4 t .. 4 t + 3 of each fourth of the tile, however the row is aligned: equal rows
  // give equal sums
#pragma unroll
  for (int j = 0; j < kEach / 4; ++j) {
    const int i = i0 + j * kScanThreads * 4 + threadIdx.x * 4;
    if (wide && i + 4 <= end) {
      const float4 v = load4(row + i);
      x[j * 4] = v.x, x[j * 4 + 1] = v.y, x[j * 4 + 2] = v.z, x[j * 4 + 3] = v.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[j * 4 + e] = i + e < end ? to_f32(row[i + e]) : -INFINITY;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kScanThreads) beam_scan_kernel(const __grid_constant__ BeamArgs a) {
  kv_enter();
  __shared__ unsigned long long held[kHeld];
  __shared__ int red[64], held_n;
  __shared__ double sums[kScanThreads / 32];
  __shared__ float tops[kScanThreads / 32];
  const int row = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int begin = blockIdx.x * a.part, end = min(a.vocab, begin + a.part);
  const T* logits = (const T*)a.logits + row * a.stride;
  const bool wide = ((uintptr_t)logits & (4 * sizeof(T) - 1)) == 0;
  BlockCount count{red, 0};
  if (threadIdx.x == 0) held_n = 0;
  float m = -INFINITY;
  double sum = 0.0;
  unsigned long long bound = 0;  // what has to be reached to be held
  bool nan = false;
  // the best a.count of what is held, moved to its front
  auto choose = [&]() {
    __syncthreads();
    const int n = held_n;
    if (n <= a.count) return;
    constexpr int E = (kHeld + kScanThreads - 1) / kScanThreads;
    unsigned long long mine[E];
#pragma unroll
    for (int j = 0; j < E; ++j) mine[j] = threadIdx.x + j * kScanThreads < n ? held[threadIdx.x + j * kScanThreads] : 0;
    bound = bound_of(a.count, bound, ~0ull - 1, count, [&](unsigned long long t) {
      int c = 0;
#pragma unroll
      for (int j = 0; j < E; ++j) c += mine[j] >= t;
      return c;
    });
    __syncthreads();
    if (threadIdx.x == 0) held_n = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < E; ++j)
      if (mine[j] >= bound && mine[j]) held[atomicAdd(&held_n, 1)] = mine[j];
    __syncthreads();
  };
#pragma unroll 1
  for (int i0 = begin; i0 < end; i0 += kTile) {
    float x[kEach];
    load_tile(logits, i0, end, wide, x);
    float top = x[0];
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      nan |= x[j] != x[j];
      top = fmaxf(top, x[j]);
    }
    if (top > m) {
      sum *= (double)expf(m - top);  // 0 where m is -inf
      m = top;
    }
    if (m != -INFINITY) {
#pragma unroll
      for (int j = 0; j < kEach; j += 4)
        sum += (double)(expf(x[j] - m) + expf(x[j + 1] - m) + (expf(x[j + 2] - m) + expf(x[j + 3] - m)));
    }
    unsigned long long best = 0;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int i = i0 + (j / 4) * kScanThreads * 4 + threadIdx.x * 4 + j % 4;
      if (i < end) best = max(best, pack(x[j], i));
    }
    if (i0 == begin) {
      // at least a.count logits reach the a.count-th of the threads' best, and at most kEach times as many
      bound = bound_of(a.count, 0, ~0ull - 1, count, [&](unsigned long long t) { return (int)(best >= t); });
    }
    if (best >= bound) {
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        const int i = i0 + (j / 4) * kScanThreads * 4 + threadIdx.x * 4 + j % 4;
        if (i >= end) continue;
        const unsigned long long p = pack(x[j], i);
        if (p >= bound) held[atomicAdd(&held_n, 1)] = p;
      }
    }
    __syncthreads();
    if (held_n > kMaxCount) choose();  // the next tile may add kTile
    __syncthreads();
  }
  choose();
  __syncthreads();
  unsigned long long* kept = a.kept + ((long long)row * a.parts + blockIdx.x) * a.count;
  for (int i = threadIdx.x; i < a.count; i += kScanThreads) kept[i] = i < held_n ? held[i] : 0;
  // the threads' sums, in an order that does not change
  float top = m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (m != -INFINITY) sum *= (double)expf(m - top);
  if (nan) sum = __longlong_as_double(0x7ff8000000000000ll);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) sums[warp] = sum, tops[warp] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
    float all = tops[0];
    for (int w = 1; w < kScanThreads / 32; ++w) all = fmaxf(all, tops[w]);
    double s = 0.0;
    for (int w = 0; w < kScanThreads / 32; ++w) s += tops[w] == -INFINITY ? sums[w] : sums[w] * (double)expf(tops[w] - all);
    a.sums[(long long)row * a.parts + blockIdx.x] = s;
    a.maxima[(long long)row * a.parts + blockIdx.x] = all;
  }
}

// ---- the choice over a batch's beams
constexpr int kPickThreads = 512, kPickChunk = 4096;

// the order of doubles as unsigned integers (no NaN comes here; the zeros alike)
__device__ __forceinline__ unsigned long long rank_key64(double v) {
  const unsigned long long b = (unsigned long long)__double_as_longlong(v == 0.0 ? 0.0 : v);
  return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ double unrank64(unsigned long long k) {
  return __longlong_as_double((long long)(k >> 63 ? k & ~(1ull << 63) : ~k));
}

struct PickShared {
  unsigned long long value[kPickChunk + kMaxCount], place[kPickChunk + kMaxCount];  // place: ~(beam * vocab + token)
  double lse[kMaxBeams];
  int red[64], n;
};

// Grid: a CTA a batch.
__global__ void __launch_bounds__(kPickThreads) beam_pick_kernel(const __grid_constant__ BeamArgs a) {
  extern __shared__ __align__(16) unsigned char smem[];
  PickShared& s = *reinterpret_cast<PickShared*>(smem);
  kv_enter();
  const int batch = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  BlockCount count{s.red, 0};
  if (threadIdx.x == 0) s.n = 0;
  for (int b = warp; b < a.beams; b += kPickThreads / 32) {
    const long long at = ((long long)batch * a.beams + b) * a.parts;
    float top = -INFINITY;
    for (int p = lane; p < a.parts; p += 32) top = fmaxf(top, a.maxima[at + p]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    double sum = 0.0;
    for (int p = lane; p < a.parts; p += 32) {
      const float m = a.maxima[at + p];
      sum += m == -INFINITY ? a.sums[at + p] : a.sums[at + p] * (double)expf(m - top);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) s.lse[b] = (double)top + log(sum);
  }
  __syncthreads();
  const long long each = (long long)a.parts * a.count, total = each * a.beams;
  unsigned long long least = 0;  // a value that a.count of what is held reach
  constexpr int E = (kPickChunk + kMaxCount + kPickThreads - 1) / kPickThreads;
#pragma unroll 1
  for (long long c0 = 0; c0 < total; c0 += kPickChunk) {
    for (int i = threadIdx.x; i < kPickChunk && c0 + i < total; i += kPickThreads) {
      const long long c = c0 + i;
      const int b = (int)(c / each), j = (int)(c - b * each);
      const float score = a.scores[(long long)batch * a.beams + b];
      const double lse = s.lse[b];
      unsigned long long p = a.kept[(long long)batch * total + c];
      double v = -INFINITY;
      int token = ~(int)(uint32_t)p;
      if (!(fabs(lse) < INFINITY) || !(score < INFINITY) || score == -INFINITY) {
        // a beam that offers nothing: of its tokens, all -inf, the first ones
        if (j >= a.count || j >= a.vocab) continue;
        token = j;
      } else {
        if (!p) continue;
        v = (double)score + ((double)unrank((uint32_t)(p >> 32)) - lse);
      }
      const unsigned long long key = rank_key64(v);
      if (key < least) continue;
      const int at = atomicAdd(&s.n, 1);
      s.value[at] = key;
      s.place[at] = ~((unsigned long long)b * a.vocab + token);
    }
    __syncthreads();
    const int n = s.n;
    if (n > a.count) {
      unsigned long long value[E], place[E];
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const int i = threadIdx.x + j * kPickThreads;
        value[j] = i < n ? s.value[i] : 0;
        place[j] = i < n ? s.place[i] : 0;
      }
      least = bound_of(a.count, least, ~0ull - 1, count, [&](unsigned long long t) {
        int k = 0;
#pragma unroll
        for (int j = 0; j < E; ++j) k += value[j] >= t;
        return k;
      });
      // of equal values at the bound, those of the lowest places
      int above = 0, reach = 0;
#pragma unroll
      for (int j = 0; j < E; ++j) above += value[j] > least, reach += value[j] >= least;
      above = count(above);
      reach = count(reach);
      unsigned long long first = 0;
      if (reach > a.count)
        first = bound_of(a.count - above, 0, ~0ull - 1, count, [&](unsigned long long t) {
          int k = 0;
#pragma unroll
          for (int j = 0; j < E; ++j) k += value[j] == least && place[j] >= t;
          return k;
        });
      __syncthreads();
      if (threadIdx.x == 0) s.n = 0;
      __syncthreads();
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (value[j] > least || (value[j] == least && value[j] && place[j] >= first)) {
          const int at = atomicAdd(&s.n, 1);
          s.value[at] = value[j];
          s.place[at] = place[j];
        }
    }
    __syncthreads();
  }
  // the chosen, each to its rank
  const int n = s.n;
  for (int i = threadIdx.x; i < n; i += kPickThreads) {
    const unsigned long long v = s.value[i], p = s.place[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += s.value[j] > v || (s.value[j] == v && s.place[j] > p);
    const long long out = (long long)batch * a.count + rank, at = (long long)~p;
    a.scores_out[out] = (float)unrank64(v);
    a.beams_out[out] = (int)(at / a.vocab);
    a.tokens_out[out] = (int)(at % a.vocab);
  }
}

struct BeamLayout {
  int parts, part;
  size_t sums, maxima, kept, bytes;
};

BeamLayout beam_layout(int rows, int vocab, int count, int sms) {
  BeamLayout L;
  // parts enough for four CTAs an SM, of whole tiles
  const int tiles = (vocab + kTile - 1) / kTile;
  long long want = (4ll * sms + rows - 1) / rows;
  if (want > tiles) want = tiles;
  const int each = (int)((tiles + want - 1) / want);
  L.part = each * kTile;
  L.parts = (tiles + each - 1) / each;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += align_up(bytes, 256);
    return here;
  };
  const size_t n = (size_t)rows * L.parts;
  L.sums = take(n * 8);
  L.maxima = take(n * 4);
  L.kept = take(n * count * 8);
  L.bytes = at;
  return L;
}

int beam_check(int dtype, int batch, int beams, int vocab, int count) {
  if (dtype != ER_DTYPE_F32 && dtype != ER_DTYPE_BF16) return fail(ER_EINVAL, "er_beam_select: logits dtype %d", dtype);
  if (batch < 0 || beams <= 0 || beams > kMaxBeams || vocab <= 0)
    return fail(ER_EINVAL, "er_beam_select: %d batches of %d beams (1 to %d), vocabulary of %d", batch, beams, kMaxBeams, vocab);
  if ((long long)batch * beams > 65535)
    return fail(ER_EINVAL, "er_beam_select: %lld rows (at most 65535)", (long long)batch * beams);
  if (count <= 0 || count > kMaxCount || count > (long long)beams * vocab)
    return fail(ER_EINVAL, "er_beam_select: count %d (1 to %d, at most beams x vocabulary)", count, kMaxCount);
  if (vocab > 0x7fff0000) return fail(ER_EINVAL, "er_beam_select: vocabulary of %d", vocab);
  return ER_OK;
}

}  // namespace
}  // namespace er

using namespace er;

extern "C" size_t er_beam_workspace_bytes(int batch, int beams, int vocab, int count) {
  int sms = 0;
  if (beam_check(ER_DTYPE_F32, batch, beams, vocab, count) || batch == 0 || device_sms(&sms)) return 0;
  return beam_layout(batch * beams, vocab, count, sms).bytes;
}

extern "C" int er_beam_select(const void* logits, int dtype, long long row_stride, const float* scores, int batch,
                              int beams, int vocab, int count, float* scores_out, int32_t* beams_out,
                              int32_t* tokens_out, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = beam_check(dtype, batch, beams, vocab, count)) return rc;
  if (row_stride < vocab) return fail(ER_EINVAL, "er_beam_select: row stride %lld shorter than the vocabulary", row_stride);
  if (batch == 0) return ER_OK;
  if (!logits || !scores || !scores_out || !beams_out || !tokens_out)
    return fail(ER_EINVAL, "er_beam_select: null pointer");
  int sms = 0;
  if (int rc = device_sms(&sms)) return rc;
  const int rows = batch * beams;
  const BeamLayout L = beam_layout(rows, vocab, count, sms);
  if (!workspace || workspace_bytes < L.bytes)
    return fail(ER_ENOSPACE, "er_beam_select: workspace %zu bytes, need %zu", workspace_bytes, L.bytes);
  if ((uintptr_t)workspace & 255) return fail(ER_EINVAL, "er_beam_select: workspace must be 256-byte aligned");
  char* ws = (char*)workspace;
  BeamArgs a = {logits, row_stride, scores, batch, beams, vocab, count, L.parts, L.part, (double*)(ws + L.sums),
                (float*)(ws + L.maxima), (unsigned long long*)(ws + L.kept), scores_out, beams_out, tokens_out};
  cudaStream_t st = (cudaStream_t)stream;
  const dim3 grid(L.parts, rows);
  int rc = dtype == ER_DTYPE_BF16
               ? kv_launch(beam_scan_kernel<__nv_bfloat16>, grid, kScanThreads, 0, false, st, "beam_scan_kernel", a)
               : kv_launch(beam_scan_kernel<float>, grid, kScanThreads, 0, false, st, "beam_scan_kernel", a);
  if (rc) return rc;
  static std::atomic<unsigned long long> allowed;
  if ((rc = allow_smem(beam_pick_kernel, (int)sizeof(PickShared), allowed))) return rc;
  return kv_launch(beam_pick_kernel, dim3(batch), kPickThreads, sizeof(PickShared), false, st, "beam_pick_kernel", a);
}
