// er_beam.cu -- beam search's choice of continuations: of every batch's
// beams x vocabulary candidates of value score + log softmax(logits)[token]
// the best `count`.
//
// The logits are read once. Within a beam the value rises with the logit, so a
// CTA that reads a part of a row keeps the part's best `count` logits (the
// other candidates cannot be chosen) beside the part's maximum and sum of
// exponentials; a second kernel joins the parts' sums and chooses among what
// was kept, by values in 64 bits: candidates of one beam keep the order of
// their logits, those of different beams compare through their beams' log-sums.
// 2 or 4 bytes a candidate and about a dozen instructions: 256 rows of 151936
// bf16 logits take 37 us (0.32 of the copy rate): 19 of instructions at the full
// rate, the barrier of a tile, and 768 CTAs for the 592 that run at once; then the
// choice over 32 batches 13 us, a chain of dependent steps in one CTA a batch, most
// of it fetching code. 4 fp32 rows: 15.5 us for both kernels (a tile a CTA; 19 as
// called), 140 rows of 50257: 33 us (700 CTAs, and a load an element).
// Exponentials, relative to a whole number that is no less than a warp's logits
// and mostly under one more than the greatest, are in 32 bits (2^-22 off, and
// |x - ref| 2^-22), and so is the sum of a thread's 16 of a tile; all sums above
// that, and what they are multiplied by when a reference rises, are in 64. A
// log-sum is good to 2^-20: beams whose values are closer may go either way.
#include "er_kv.cuh"
#include "er_ptx.cuh"

namespace er {

namespace {

constexpr int kScanThreads = 256, kEach = 16, kTile = kScanThreads * kEach;  // logits a tile
constexpr int kMaxCount = 128, kMaxBeams = 1024;
constexpr int kHeld = kTile + kScanThreads;  // what a CTA may hold before it has to choose

struct BeamArgs {
  const void* logits;
  long long stride;
  const float* scores;
  int batch, beams, vocab, count;
  int parts, part;  // of a row, and logits of each (a multiple of the tile)
  double* sums;     // [rows][parts] of exponentials, relative to e^refs
  float* refs;      // [rows][parts]
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

// A bound that at least `want` of the block's keys reach and, where that can be, at most `enough` (has(t): how many
// of the thread's keys are >= t), by halving. `least`: one that `want` reach; `most`: none above it is reached by as many.
template <typename Has>
__device__ __forceinline__ unsigned long long bound_of(int want, int enough, unsigned long long least,
                                                       unsigned long long most, BlockCount& count, Has has) {
  while (least < most) {
    const unsigned long long mid = least + (most - least) / 2 + 1;
    const int n = count(has(mid));
    if (n >= want && n <= enough) return mid;
    if (n > want)
      least = mid;
    else
      most = mid - 1;
  }
  return least;
}

// Appends the keys of the threads that have one to a list in shared memory, a warp at a time.
__device__ __forceinline__ int place_of(bool mine, int* n) {
  const uint32_t all = __ballot_sync(0xffffffffu, mine);
  int base = 0;
  if ((threadIdx.x & 31) == 0 && all) base = atomicAdd(n, __popc(all));
  return __shfl_sync(0xffffffffu, base, 0) + __popc(all & ((1u << (threadIdx.x & 31)) - 1));
}

// Sixteen logits of a tile, runs of kRun: thread t has runs t, t + 256, ... however the row is aligned, so that equal
// rows give equal sums. Those behind the end are -inf.
template <typename T>
struct Logits {
  static constexpr int kRun = 16 / (int)sizeof(T), kRuns = kEach / kRun;
  uint4 raw[kRuns];

  __device__ __forceinline__ static int at(int j) { return (j / kRun) * kScanThreads * kRun + threadIdx.x * kRun + j % kRun; }
  __device__ __forceinline__ void load(const T* row, int i0, int end, bool wide) {
#pragma unroll
    for (int r = 0; r < kRuns; ++r) {
      const int i = i0 + at(r * kRun);
      if (wide && i + kRun <= end) {
        raw[r] = __ldg(reinterpret_cast<const uint4*>(row + i));
      } else {
        uint32_t h[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (sizeof(T) == 4) {
            h[e] = i + e < end ? __float_as_uint(row[i + e]) : 0xff800000u;
          } else {
            const uint32_t lo = i + 2 * e < end ? __bfloat16_as_ushort(row[i + 2 * e]) : 0xff80u;
            const uint32_t hi = i + 2 * e + 1 < end ? __bfloat16_as_ushort(row[i + 2 * e + 1]) : 0xff80u;
            h[e] = lo | hi << 16;
          }
        }
        raw[r] = make_uint4(h[0], h[1], h[2], h[3]);
      }
    }
  }
  __device__ __forceinline__ void floats(float (&x)[kEach]) const {
#pragma unroll
    for (int r = 0; r < kRuns; ++r) {
      const uint32_t h[4] = {raw[r].x, raw[r].y, raw[r].z, raw[r].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (sizeof(T) == 4) {
          x[r * kRun + e] = __uint_as_float(h[e]);
        } else {
          x[r * kRun + 2 * e] = __uint_as_float(h[e] << 16);
          x[r * kRun + 2 * e + 1] = __uint_as_float(h[e] & 0xffff0000u);
        }
      }
    }
  }
};

// What a sum is multiplied by when its reference rises by a whole number: a power of 1/e, within 2^-46. (As an
// exponential in 32 bits it is 2^-22 off, and rows that rise with every tile gather that: 123 tiles 7 x 2^-21.)
__device__ __forceinline__ double relative_to(double sum, float from, float to) {
  const float by = to - from;
  if (!(by > 0.f)) return sum;  // NaN: none of the two is finite
  double power = 0.36787944117144233;
  // e^-63 is less than the last bit of any sum; mostly 1 or 2
  for (int n = by < 63.f ? (int)by : 63; n; n >>= 1, power *= power)
    if (n & 1) sum *= power;
  return sum;
}

// the greatest of the warp's (NaN where that is what a lane has)
__device__ __forceinline__ float warp_max(float x) {
  auto order = [](int b) { return b ^ (b >> 31 & 0x7fffffff); };
  return __int_as_float(order(__reduce_max_sync(0xffffffffu, order(__float_as_int(x)))));
}

// Of every logit: a maximum, a subtraction, a product, an exponential and a sum; whether it can be among the best is
// asked of a thread's greatest, and only a thread that has one looks again. Sums of 16 go to 64 bits.
template <typename T>
__global__ void __launch_bounds__(kScanThreads, 4) beam_scan_kernel(const __grid_constant__ BeamArgs a) {
  kv_enter();
  __shared__ unsigned long long held[kHeld];
  __shared__ int red[64], held_n;
  __shared__ uint32_t warp_least[kScanThreads / 32];
  __shared__ double sums[kScanThreads / 32];
  __shared__ float refs[kScanThreads / 32];
  const int row = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int begin = blockIdx.x * a.part, end = begin + min(a.vocab - begin, a.part);
  const T* logits = (const T*)a.logits + row * a.stride;
  const bool wide = ((uintptr_t)logits & 15) == 0;
  BlockCount count{red, 0};
  Logits<T> next;
  next.load(logits, begin, end, wide);
  if (threadIdx.x == 0) held_n = 0;
  float m = -INFINITY, ref = -INFINITY;  // the thread's greatest logit, and what the warp's sums are relative to
  double sum = 0.0;
  unsigned long long bound = 0;  // what has to be reached to be held
  float least = -INFINITY;       // its logit (what is not below it may be held)
  int most_held = 0;             // the same in all threads, and no less than is held
  // the best of what is held, a.count to kScanThreads of them, moved to its front
  auto choose = [&]() {
    __syncthreads();
    const int n = held_n;
    if (n <= kScanThreads) return;
    bound = bound_of(a.count, kScanThreads, bound, ~0ull - 1, count, [&](unsigned long long t) {
      int c = 0;
      for (int i = threadIdx.x; i < n; i += kScanThreads) c += held[i] >= t;
      return c;
    });
    least = unrank((uint32_t)(bound >> 32));
    if (threadIdx.x == 0) held_n = 0;
    __syncthreads();
    for (int i0 = 0; i0 < n; i0 += kScanThreads) {
      // entries in front of i0 were read before, and no more of them than of those can have been kept
      const unsigned long long mine = i0 + (int)threadIdx.x < n ? held[i0 + threadIdx.x] : 0;
      __syncthreads();
      const bool take = mine && mine >= bound;
      const int at = place_of(take, &held_n);
      if (take) held[at] = mine;
      __syncthreads();
    }
  };
#pragma unroll 1
  for (int tile = 0; begin + tile * kTile < end; ++tile) {
    const int i0 = begin + tile * kTile;
    float x[kEach];
    next.floats(x);
    if (i0 + kTile < end) next.load(logits, i0 + kTile, end, wide);
    float top = x[0];
#pragma unroll
    for (int j = 1; j < kEach; ++j) top = fmaxf(top, x[j]);
    m = fmaxf(m, top);
    const float warp_top = warp_max(top);
    if (warp_top > ref) {
      const float up = ceilf(warp_top);
      if (ref != -INFINITY) sum = relative_to(sum, ref, up);  // 0, or NaN, where it is
      ref = up;
    }
    // a warp whose logits are all -inf, or NaN among them, so far: its sums stay 0, or become NaN
    const float from = ref == -INFINITY ? 0.f : ref;
    const uint64_t off = pack2(-from, -from), unit = pack2(1.44269504f, 1.44269504f);
    uint64_t part[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < kEach; j += 2) {
      float u, v;  // e^(x - ref): within 2^-22 and |x - ref| 2^-22 of it
      unpack2(fma2(add2(pack2(x[j], x[j + 1]), off), unit, 0), u, v);
      part[j / 2 & 1] = add2(part[j / 2 & 1], pack2(ex2(u), ex2(v)));
    }
    float even, odd;
    unpack2(add2(part[0], part[1]), even, odd);
    sum += (double)(even + odd);
    if ((tile & (tile - 1)) == 0) {
      // A bound from the threads' greatest so far, renewed as the tiles double: as many of each warp's as make a.count
      // of the block's reach the least of what the warps' do.
      uint32_t key = begin + Logits<T>::at(0) < end ? rank_key(m) : 0u, r = 0;
      for (int k = 0; k < a.count; k += kScanThreads / 32) {
        r = __reduce_max_sync(0xffffffffu, key);
        const uint32_t who = __ballot_sync(0xffffffffu, key == r);
        if (lane == __ffs(who) - 1) key = 0;
      }
      if (lane == 0) warp_least[warp] = r;
      __syncthreads();
      r = warp_least[0];
      for (int w = 1; w < kScanThreads / 32; ++w) r = min(r, warp_least[w]);
      const unsigned long long now = (unsigned long long)r << 32;
      if (now > bound) bound = now, least = unrank(r);
    }
    bool look = !(top < least);
    const int lookers = __syncthreads_count(look) * kEach;  // what was held before is there, too
    if (most_held + lookers > kHeld) {
      most_held = held_n;
      __syncthreads();
      if (most_held + lookers > kHeld) {
        choose();
        most_held = kScanThreads;
        look = !(top < least);
      }
    }
    most_held += lookers;
    if (look) {
      uint32_t which = 0;
#pragma unroll
      for (int j = 0; j < kEach; ++j) which |= (uint32_t)!(x[j] < least) << j;
      for (; which; which &= which - 1) {  // few: read again
        const int i = i0 + Logits<T>::at(__ffs(which) - 1);
        if (i >= end) continue;
        const unsigned long long p = pack((float)logits[i], i);
        if (p >= bound) held[atomicAdd(&held_n, 1)] = p;
      }
    }
  }
  choose();
  // the best of them, a thread each, to its rank (no two keys are alike)
  unsigned long long* kept = a.kept + ((long long)row * a.parts + blockIdx.x) * a.count;
  const int n = held_n;
  const unsigned long long mine = (int)threadIdx.x < n ? held[threadIdx.x] : 0;
  if (__any_sync(0xffffffffu, mine && mine >= bound)) {
    int rank = mine && mine >= bound ? 0 : kHeld;
#pragma unroll 8
    for (int i = 0; i < n; ++i) rank += held[i] > mine;
    if (rank < a.count) kept[rank] = mine;
  }
  if ((int)threadIdx.x >= n && (int)threadIdx.x < a.count) kept[threadIdx.x] = 0;
  // the threads' sums, in an order that does not change
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) sums[warp] = sum, refs[warp] = ref;
  __syncthreads();
  if (threadIdx.x == 0) {
    float all = refs[0];
    for (int w = 1; w < kScanThreads / 32; ++w) all = fmaxf(all, refs[w]);
    double s = 0.0;
    for (int w = 0; w < kScanThreads / 32; ++w) s += refs[w] == -INFINITY ? sums[w] : relative_to(sums[w], refs[w], all);
    a.sums[(long long)row * a.parts + blockIdx.x] = s;
    a.refs[(long long)row * a.parts + blockIdx.x] = all;
  }
}

// ---- the choice over a batch's beams
constexpr int kPickThreads = 512, kPickEach = 4, kPickChunk = kPickThreads * kPickEach, kFew = 128;

// the order of doubles as unsigned integers (no NaN comes here; the zeros alike)
__device__ __forceinline__ unsigned long long rank_key64(double v) {
  const unsigned long long b = (unsigned long long)__double_as_longlong(v == 0.0 ? 0.0 : v);
  return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ double unrank64(unsigned long long k) {
  return __longlong_as_double((long long)(k >> 63 ? k & ~(1ull << 63) : ~k));
}

struct PickShared {
  // candidates, by what they are ordered by: the value, kMaxBeams - 1 - beam, the logit's rank and ~token
  unsigned long long value[kPickChunk + kMaxCount], logit[kPickChunk + kMaxCount];
  uint16_t beam[kPickChunk + kMaxCount];
  double lse[kMaxBeams];
  int red[64], n;
  uint32_t warp_least[kPickThreads / 32];
};

// Grid: a CTA a batch. It goes over what was kept kPickChunk at a time: those that may be among the best join the best
// so far in shared memory, and the best of them are found by a bound on their values, then by their ranks.
__global__ void __launch_bounds__(kPickThreads) beam_pick_kernel(const __grid_constant__ BeamArgs a) {
  extern __shared__ __align__(16) unsigned char smem[];
  PickShared& s = *reinterpret_cast<PickShared*>(smem);
  kv_enter();
  const int batch = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int each = a.parts * a.count;  // of a beam
  const long long total = (long long)each * a.beams;
  unsigned long long kept[kPickEach];
  auto fetch = [&](long long c0) {
#pragma unroll
    for (int i = 0; i < kPickEach; ++i) {
      const long long c = c0 + i * kPickThreads + threadIdx.x;
      kept[i] = c < total ? a.kept[(long long)batch * total + c] : 0;
    }
  };
  fetch(0);
  BlockCount count{s.red, 0};
  if (threadIdx.x == 0) s.n = 0;
  const long long row0 = (long long)batch * a.beams;
  for (int b = warp; b < a.beams; b += kPickThreads / 32) {
    const long long at = (row0 + b) * a.parts;
    float top = -INFINITY;
    for (int p = lane; p < a.parts; p += 32) top = fmaxf(top, a.refs[at + p]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    double sum = 0.0;
    for (int p = lane; p < a.parts; p += 32) {
      const float ref = a.refs[at + p];
      sum += ref == -INFINITY ? a.sums[at + p] : relative_to(a.sums[at + p], ref, top);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) s.lse[b] = (double)top + log(sum);
  }
  __syncthreads();
  // Of the threads' greatest values (their upper words), as many of each warp's as make a.count of the block's reach the
  // least of what the warps' do.
  auto bound_above = [&](uint32_t key) {
    uint32_t r = 0;
    for (int k = 0; k < a.count; k += kPickThreads / 32) {
      r = __reduce_max_sync(0xffffffffu, key);
      const uint32_t who = __ballot_sync(0xffffffffu, key == r);
      if (lane == __ffs(who) - 1) key = 0;
    }
    if (lane == 0) s.warp_least[warp] = r;
    __syncthreads();
    return (unsigned long long)__reduce_min_sync(0xffffffffu, s.warp_least[lane & (kPickThreads / 32 - 1)]) << 32;
  };
  unsigned long long least = 0;  // a value that a.count of what is held reach
  constexpr int E = kPickEach + 1;
#pragma unroll 1
  for (long long c0 = 0; c0 < total; c0 += kPickChunk) {
    unsigned long long key[kPickEach], logit[kPickEach];
    int beam[kPickEach];
    uint32_t best = 0;
#pragma unroll
    for (int i = 0; i < kPickEach; ++i) {
      const long long c = c0 + i * kPickThreads + threadIdx.x;
      bool take = c < total;
      logit[i] = key[i] = 0;
      beam[i] = 0;
      if (take) {
        const int b = (int)(c >> 32 ? c / each : (uint32_t)c / (uint32_t)each), j = (int)(c - (long long)b * each);
        const float score = a.scores[row0 + b];
        const double lse = s.lse[b];
        const unsigned long long p = kept[i];
        double v = -INFINITY;
        logit[i] = p;
        beam[i] = kMaxBeams - 1 - b;
        if (!(fabs(lse) < INFINITY) || !(score < INFINITY) || score == -INFINITY) {
          // a beam that offers nothing: of its tokens, all -inf, the first ones
          take = j < a.count && j < a.vocab;
          logit[i] = (uint32_t)~j;
        } else {
          take = p != 0;
          v = (double)score + ((double)unrank((uint32_t)(p >> 32)) - lse);
        }
        if (take) key[i] = rank_key64(v);
      }
      best = max(best, (uint32_t)(key[i] >> 32));
    }
    least = max(least, bound_above(best));
#pragma unroll
    for (int i = 0; i < kPickEach; ++i) {
      const bool take = key[i] && key[i] >= least;
      const int at = place_of(take, &s.n);
      if (take) s.value[at] = key[i], s.logit[at] = logit[i], s.beam[at] = (uint16_t)beam[i];
    }
    if (c0 + kPickChunk < total) fetch(c0 + kPickChunk);
    __syncthreads();
    const int n = s.n;
    const int enough = c0 + kPickChunk < total ? a.count : a.count + kFew;
    if (n > enough) {  // a few are ranked as they are
      unsigned long long value[E], logit[E];
      int beam[E];
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const int i = threadIdx.x + j * kPickThreads;
        value[j] = i < n ? s.value[i] : 0;
        logit[j] = i < n ? s.logit[i] : 0;
        beam[j] = i < n ? s.beam[i] : 0;
      }
      auto reaching = [&](unsigned long long t) {
        int k = 0;
#pragma unroll
        for (int j = 0; j < E; ++j) k += value[j] >= t;
        return k;
      };
      least = bound_of(a.count, enough, least, ~0ull - 1, count, reaching);
      // of equal values at the bound, where they are many, those of the lowest beams, of the last of these the greatest logits
      int above = 0, reach = 0;
#pragma unroll
      for (int j = 0; j < E; ++j) above += value[j] > least, reach += value[j] >= least;
      above = count(above);
      reach = count(reach);
      int last = -1;
      unsigned long long first = 0;
      if (above < a.count && reach > enough) {
        int want = a.count - above, before = 0;
        last = (int)bound_of(want, want, 0, kMaxBeams - 1, count, [&](unsigned long long t) {
          int k = 0;
#pragma unroll
          for (int j = 0; j < E; ++j) k += value[j] == least && beam[j] >= (int)t;
          return k;
        });
#pragma unroll
        for (int j = 0; j < E; ++j) before += value[j] == least && beam[j] > last;
        want -= count(before);
        first = bound_of(want, want, 0, ~0ull - 1, count, [&](unsigned long long t) {
          int k = 0;
#pragma unroll
          for (int j = 0; j < E; ++j) k += value[j] == least && beam[j] == last && logit[j] >= t;
          return k;
        });
      }
      __syncthreads();
      if (threadIdx.x == 0) s.n = 0;
      __syncthreads();
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const bool take = value[j] > least ||
                          (value[j] == least && value[j] && (beam[j] > last || (beam[j] == last && logit[j] >= first)));
        const int at = place_of(take, &s.n);
        if (take) s.value[at] = value[j], s.logit[at] = logit[j], s.beam[at] = (uint16_t)beam[j];
      }
    }
    __syncthreads();
  }
  // the best of them, each to its rank
  const int n = s.n;
  for (int i = warp; i < n; i += kPickThreads / 32) {
    const unsigned long long v = s.value[i], p = s.logit[i];
    const int b = s.beam[i];
    int rank = 0;
#pragma unroll 4
    for (int j = lane; j < n; j += 32) {
      const unsigned long long u = s.value[j];
      rank += u > v || (u == v && (s.beam[j] > b || (s.beam[j] == b && s.logit[j] > p)));
    }
    rank = __reduce_add_sync(0xffffffffu, rank);
    if (rank >= a.count || lane) continue;
    const long long out = (long long)batch * a.count + rank;
    a.scores_out[out] = (float)unrank64(v);
    a.beams_out[out] = kMaxBeams - 1 - b;
    a.tokens_out[out] = (int)~(uint32_t)p;
  }
}

struct BeamLayout {
  int parts, part;
  size_t sums, refs, kept, bytes;
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
  L.refs = take(n * 4);
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
                (float*)(ws + L.refs), (unsigned long long*)(ws + L.kept), scores_out, beams_out, tokens_out};
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
