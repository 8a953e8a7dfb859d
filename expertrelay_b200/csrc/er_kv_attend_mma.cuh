// er_kv_attend_mma.cuh -- attention over a paged key-value cache on the tensor cores.
//
// One key and its value (2 d elements) take part in 4 d G flop, so the cache
// streams from memory while the arithmetic waits, as long as no lane touches
// each value G times: a warp multiplies 16 keys with the group's queries by
// m16n8 matrix instructions, keys (scores) or channels (values) along m and
// up to 8 queries along n, which pads a group of one to 8 columns for nothing
// but idle tensor cores. tcgen05 would take 64 rows of keys at the least, its
// operands and results through tensor memory; a chunk that one warp loads,
// multiplies and drops needs no barrier between warps at all.
//
//   scores^T [16 keys x 8 queries]  = K [16 x d] . Q^T
//   out^T    [d x 8 queries]       += V^T [d x 16 keys] . P^T [16 keys x 8 queries]
//
// K comes by ldmatrix, Q^T lies in shared memory in the instructions' order,
// and the scores' accumulator turns into P^T by 8x8 transposes (movmatrix).
//
// Numbers. bf16 caches (m16n8k16, V by ldmatrix.trans): bf16 has 8 bits, fp32
// 24; fp32 queries enter as the exact sum of three bf16 parts, and so do the
// weights. Parts are cut, not rounded, so that they share the sign of the whole
// and an infinite key or value stays infinite. fp32 caches (m16n8k8, tf32 with
// 11 bits): every operand is its leading 11 bits and the rest (11 more), and of
// the products all but rest times rest (2^-21 of the whole at the most, of
// either sign) are taken: with that product too, 344 us became 363 and 482
// became 540 below. Where a key or value that is seen is infinite, the result is
// infinite or NaN. The tensor cores cut their sums (they do not round), so a
// chunk's products are added up there and the running sum over the chunks in
// rounded fp32, whatever the result's type. (With weights of two parts and the
// sums left in the tensor cores, bf16 results took 166 us in place of 170 below
// and were 3 to 4.5 10^-6 off before their rounding, now 1 to 5 10^-7: of 400000
// outputs 0.35 % were rounded to the wrong side, 0.02 % are.)
//
// Measured (16 rows of 16000 positions, 8 key heads, head_dim 128, pages of 16;
// at the rate of a copy bf16 pages take 161 us, fp32 pages 322): bf16 pages and
// queries, 4 queries a key head 170 us, 16 queries 236; fp32 queries 183 and
// 262; fp32 pages 344 and 482. With 4 queries memory bounds it; with 16 the
// chain of a tile's steps in a warp does, and the rescaling and exponentials of
// twice as many columns.
#pragma once

#include <type_traits>

#include "er_kv_attend.cuh"

namespace er {

namespace {

__device__ __forceinline__ void ldsm(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The leading bf16 part of two floats (their upper halves), packed; x, y
// become what is left.
__device__ __forceinline__ uint32_t cut2(float& x, float& y) {
  const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
  x -= __uint_as_float(a & 0xffff0000u);
  y -= __uint_as_float(b & 0xffff0000u);
  return __byte_perm(a, b, 0x7632);
}

// A query as three bf16 parts (bits) whose sum it is exactly. A part that is
// zero where the query is not takes the least value of its sign (2^-133):
// times an infinite key it has to stay infinite, and beside a finite one it
// vanishes.
__device__ __forceinline__ void query_parts(float x, uint32_t (&p)[3]) {
  const uint32_t tiny = __float_as_uint(x) >> 31 << 15 | 1u;
  const bool finite = fabsf(x) < INFINITY;
  p[0] = x != x ? 0x7fc0u : __float_as_uint(x) >> 16;
  float rest = finite ? x - __uint_as_float(p[0] << 16) : 0.f;
  p[1] = __float_as_uint(rest) >> 16;
  rest -= __uint_as_float(p[1] << 16);
  p[2] = __float_as_uint(rest) >> 16;
#pragma unroll
  for (int i = 0; i < 3; ++i)
    if ((p[i] & 0x7fff) == 0 && x != 0.f) p[i] = tiny;
}

__device__ __forceinline__ void mma_tf32(float (&c)[4], const float (&a)[4], float b0, float b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(__float_as_uint(a[0])), "r"(__float_as_uint(a[1])), "r"(__float_as_uint(a[2])), "r"(__float_as_uint(a[3])),
        "r"(__float_as_uint(b0)), "r"(__float_as_uint(b1)));
}
// x, such that its leading 11 bits (all that the tensor cores look at) are x rounded
__device__ __forceinline__ float round_tf32(float x) { return __uint_as_float(__float_as_uint(x) + 0x1000u); }
// the leading 11 bits of x; x becomes the rest
__device__ __forceinline__ float cut_tf32(float& x) {
  const float hi = __uint_as_float(__float_as_uint(x) & 0xffffe000u);
  x -= hi;
  return hi;
}

constexpr int kMergeHeads = 4;  // queries whose pieces the warps exchange at a time

// A CTA's shape for a cache of TC, queries and results of TQ, head_dim padded
// to DP, NT tiles of 8 queries. What bounds a warp is the chain of a tile (wait,
// scores, maximum, exponentials, products), so what carries it are warps
// enough, as many on each of the SM's four schedulers, and registers enough for
// each (8 warps of 255, 12 of 168); 96 to 192 KB under way on an SM come with
// that. Times of 16 rows, 8 key heads, 4 queries each, over 1.05 GB of keys and
// values (rows of 512 bytes and more: 2.1 GB):
//   bf16 rows of 128 bytes: 12 warps of 32 keys, two stages (8 warps: 194 us, 167)
//     256 bytes: 8 warps of 16 keys, two stages (170 us; one stage of 32 keys 176);
//       of 32 keys and one stage where the queries have parts or two tiles
//       (16 queries a key head: 225 us with 16 keys and two stages, 211)
//     512 bytes: 8 warps of one stage (4 of three: 350 us, 314; 7 of one: 323)
//   (pairs with 167, 211 and 314 are of weights in two parts; in three, the ones
//   taken are at 179, 236 and 321)
//   fp32 rows of 256 bytes: 12 warps of one stage, 8 of two for two tiles (206 us, 193)
//     512 bytes: 8 warps of one stage (6 of two: 404 us, 345; 10 of one, registers short: 396)
//     1024 bytes: 5 warps of one stage, all that fits (3 of two: 723 us, 443)
template <typename TC, typename TQ, int DP, int NT>
struct Mma {
  static constexpr bool kBf16 = sizeof(TC) == 2;
  // parts of a query and of a weight (fp32 caches: leading bits and rest)
  static constexpr int QS = !kBf16 ? 2 : sizeof(TQ) == 2 ? 1 : 3, PS = kBf16 ? 3 : 2;
  static constexpr int kRow = DP * (int)sizeof(TC);  // bytes of a key in shared memory
  static constexpr bool kParts = NT * QS > 1;
  static constexpr int kKeys = kBf16 && (kRow == 128 || (kRow == 256 && kParts)) ? 32 : 16;  // keys a warp takes at a time
  static constexpr int kChunkBytes = kKeys * kRow;
  static constexpr int kWarps = kBf16 ? (kRow == 128 ? 6 : kRow == 256 ? 4 : 8)
                                      : kRow == 256 ? (NT == 1 ? 6 : 4) : kRow == 512 ? (NT == 1 ? 4 : 8) : 5;
  static constexpr int kStages = kBf16 ? (kRow == 128 || (kRow == 256 && !kParts) ? 2 : 1) : kRow == 256 && NT == 2 ? 2 : 1;
  static constexpr int kRing = kWarps * kStages * 2 * kChunkBytes;
  static constexpr int kKSteps = kBf16 ? DP / 16 : DP / 8;  // matrix products along the channels of the scores
  static constexpr int kQuery = kKSteps * QS * NT * 32 * 8;
  static constexpr int kSmem = kRing + kQuery + kWarps * kMergeHeads * DP * 4 + kWarps * NT * 8 * 2 * 4;
  static constexpr int kPerSm = 2 * (kSmem + 3584) <= 228 * 1024 ? 2 : 1;
  static_assert(kSmem + 3584 <= 228 * 1024, "fits an SM");
  static_assert(NT * 8 * (DP + 2) * 4 <= kRing, "a cluster's piece fits the ring");
};

// Byte offset of the 16-byte column `col` of row `row`: columns permuted
// within each 128 bytes by the row, so that 8 rows' copies of one column lie
// in 8 different bank groups.
template <int ROW>
__device__ __forceinline__ int swz(int row, int col) {
  return row * ROW + ((col ^ (row & 7)) << 4);
}

}  // namespace

// DP: head_dim padded to 64, 128 or 256; NT: tiles of 8 queries. WHOLE:
// page_size is a multiple of 8. CLUSTER: a cluster per unit.
template <typename TC, typename TQ, int DP, int NT, bool WHOLE, bool CLUSTER>
__global__ void __launch_bounds__(Mma<TC, TQ, DP, NT>::kWarps * 32, Mma<TC, TQ, DP, NT>::kPerSm)
    kv_attend_kernel(const __grid_constant__ AttendArgs a) {
  using C = Mma<TC, TQ, DP, NT>;
  constexpr int S = C::kStages, KEYS = C::kKeys, KB = KEYS / 16, KS = C::kKSteps, QS = C::QS, PS = C::PS, W = C::kWarps;
  constexpr int MT = DP / 16;  // tiles of 16 channels
  // Over 1024-byte rows the products of the last quarter stand behind a branch
  // of their own (256 channels: 550 -> 443 us, the code then keeps to its
  // registers; 192: 551 -> 380). Elsewhere that branch cost 1 .. 20 %.
  constexpr int DP1 = !C::kBf16 && DP == 256 ? 192 : DP, KS1 = KS * DP1 / DP, MT1 = MT * DP1 / DP;
  constexpr bool BF = C::kBf16;
  extern __shared__ __align__(128) char sm[];
  __shared__ RunScratch scratch;
  __shared__ int spoiled;
  __shared__ StageInfo info[W][S];
  const int d = a.kv.d, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  char* ring = sm + warp * S * 2 * C::kChunkBytes;
  uint2* qf = reinterpret_cast<uint2*>(sm + C::kRing);                   // [KS][QS][NT][32]
  float* merge = reinterpret_cast<float*>(sm + C::kRing + C::kQuery);    // [warps][kMergeHeads][DP]
  float* ml = merge + W * kMergeHeads * DP;                              // [warps][NT * 8][2]
  const int cols = d * (int)sizeof(TC) / 16;                             // 16-byte columns of a row
  constexpr int WIDE = C::kRow / 16 < 32 ? C::kRow / 16 : 32, CW = C::kRow / 16 / WIDE;  // lanes a row, columns a lane
  constexpr int KG = 32 / WIDE;
  const int col = lane % WIDE, kg = lane / WIDE;

  if (d < DP) {  // the columns behind head_dim stay zero
    for (int i = lane; i < S * 2 * C::kChunkBytes / 16; i += 32)
      *reinterpret_cast<uint4*>(ring + i * 16) = make_uint4(0, 0, 0, 0);
    __syncwarp();
  }
  kv_enter();
  // a cluster's CTA leaves its piece where its ring was
  float *piece_ml = reinterpret_cast<float*>(sm), *piece_o = piece_ml + NT * 8 * 2;
  const Run run = CLUSTER ? kv_cluster_run(a) : kv_run(a, scratch);
  if (run.left == 0) {
    if (CLUSTER) {
      __syncthreads();  // the ring's zeros are written
      for (int i = threadIdx.x; i < NT * 8 * (DP + 2); i += W * 32) piece_ml[i] = i < NT * 16 && !(i & 1) ? -INFINITY : 0.f;
      kv_cluster_join<TQ>(a, run, NT * 8, piece_ml, piece_o, DP);
    }
    return;
  }
  long long left = run.left, begin = run.begin;
  Walk<WHOLE, KEYS> walk(a, run);

  float m[NT][2], l[NT][2], o[MT][NT][4];
  bool fresh = true, bad = false;
  int st = 0, first_t = 0, live_g = 0, filled = 0;
  // One loop fills the ring (S steps), then takes a stage and fills it again:
  // each piece of code stands once, since a short launch waits for its
  // instructions as it does for its data.
#pragma unroll 1
  for (;;) {
    const bool work = filled == S;
    StageInfo now = {};
    if (work) {
      if (S == 1) __syncwarp();  // lane 0 has just written it; of more stages, before the last tile's __syncwarp
      now = info[warp][st];
    }
    // a new unit: its queries in the matrix instructions' order (the first
    // unit's before the ring is filled, while its pages are looked up)
    if (fresh && (work || filled == 0)) {
      if (!work) now = walk.info(a, 0, 0, NT * 8);
      fresh = false;
      bad = false;
      first_t = now.t;
      live_g = min(NT * 8, a.group - now.g0);
      const TQ* qr = (const TQ*)a.q + (long long)now.row * a.q_stride + (long long)(now.head * a.group + now.g0) * d;
#pragma unroll 2
      for (int i = threadIdx.x; i < KS * NT * 32; i += W * 32) {
        const int ln = i % 32, nt = i / 32 % NT, ks = i / (32 * NT), g = nt * 8 + ln / 4;
        // the lane's channels of query g: (c, c + 1, c + 8, c + 9) or (c, c + 4)
        const int c0 = BF ? ks * 16 + ln % 4 * 2 : ks * 8 + ln % 4;
        uint2* to = qf + (ks * QS * NT + nt) * 32 + ln;
        if constexpr (BF) {
          uint32_t p[4][QS];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int cc = c0 + (e & 1) + (e >> 1) * 8;
            const bool on = g < live_g && cc < d;
            if constexpr (QS == 1)
              p[e][0] = on ? (uint32_t)reinterpret_cast<const uint16_t*>(qr)[g * d + cc] : 0u;
            else
              query_parts(on ? to_f32(qr[g * d + cc]) : 0.f, p[e]);
          }
#pragma unroll
          for (int i2 = 0; i2 < QS; ++i2)
            to[i2 * NT * 32] = make_uint2(p[0][i2] | p[1][i2] << 16, p[2][i2] | p[3][i2] << 16);
        } else {
          float x[2], hi[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int cc = c0 + e * 4;
            x[e] = g < live_g && cc < d ? to_f32(qr[g * d + cc]) : 0.f;
            // leading bits rounded, so that the rest has either sign and what the
            // products leave out (rest times rest) has no mean; cut where that overflows
            const float near = __uint_as_float(__float_as_uint(round_tf32(x[e])) & 0xffffe000u);
            if (fabsf(near) < INFINITY && fabsf(x[e]) < INFINITY) {
              hi[e] = near;
              x[e] = round_tf32(x[e] - near);
            } else {
              hi[e] = cut_tf32(x[e]);
              if (!(fabsf(hi[e]) < INFINITY)) x[e] = 0.f;
            }
          }
          to[0] = make_uint2(__float_as_uint(hi[0]), __float_as_uint(hi[1]));
          to[NT * 32] = make_uint2(__float_as_uint(x[0]), __float_as_uint(x[1]));
        }
      }
      if (threadIdx.x == 0) spoiled = 0;
      __syncthreads();
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        m[nt][0] = m[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
        for (int k = 0; k < MT; ++k) o[k][nt][0] = o[k][nt][1] = o[k][nt][2] = o[k][nt][3] = 0.f;
      }
    }
    if (work) {
      copy_wait<S - 1>();
      __syncwarp();
      if (now.bad) bad = true;
      if (now.keys) {
        const uint32_t kc = smem_addr(ring + st * 2 * C::kChunkBytes), vc = kc + C::kChunkBytes;
        const int mi = lane / 8, mr = lane % 8;  // the 8x8 matrix and its row that this lane addresses
        // Two or three chains of products: their latencies overlap, and each is
        // summed over fewer steps (the parts below the leading ones in the
        // last). With 32 keys the key blocks are chains of their own.
        constexpr int CH = !BF ? 3 : KB == 1 || QS > 1 ? 2 : 1;
        float s2[KB][CH][NT][4];
#pragma unroll
        for (int i = 0; i < KB * CH * NT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) s2[i / (CH * NT)][i / NT % CH][i % NT][e] = 0.f;
        auto score = [&](int ks) {
#pragma unroll
          for (int kb = 0; kb < KB; ++kb) {
            uint32_t kf[4];
            ldsm(kf, kc + swz<C::kRow>(kb * 16 + (mi & 1) * 8 + mr, ks * 2 + (mi >> 1)));
            if constexpr (BF) {
#pragma unroll
              for (int p = 0; p < QS; ++p)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                  const uint2 b = qf[((ks * QS + p) * NT + nt) * 32 + lane];
                  mma(s2[kb][CH == 1 ? 0 : QS == 1 ? ks & 1 : p > 0][nt], kf, b.x, b.y);
                }
            } else {
              float lo[4], hi[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                lo[e] = __uint_as_float(kf[e]);
                hi[e] = cut_tf32(lo[e]);
                lo[e] = round_tf32(lo[e]);  // cut, it would lower every score by about 2^-23 of it
              }
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                const uint2 bh = qf[(ks * QS * NT + nt) * 32 + lane], bl = qf[((ks * QS + 1) * NT + nt) * 32 + lane];
                mma_tf32(s2[kb][CH - 1][nt], lo, __uint_as_float(bh.x), __uint_as_float(bh.y));
                mma_tf32(s2[kb][CH - 1][nt], hi, __uint_as_float(bl.x), __uint_as_float(bl.y));
                mma_tf32(s2[kb][ks & (CH / 2)][nt], hi, __uint_as_float(bh.x), __uint_as_float(bh.y));
              }
            }
          }
        };
#pragma unroll(KS1 <= 16 ? KS1 : 8)
        for (int ks = 0; ks < KS1; ++ks) score(ks);
        if (KS1 < KS && d > DP1) {
#pragma unroll
          for (int ks = KS1; ks < KS; ++ks) score(ks);
        }
        // p: [kb][nt][e]: key kb 16 + lane / 4 + 8 (e / 2), query 2 (lane % 4) + e % 2
        float high[NT][2], p[KB][NT][4];
        bool moved = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const bool on = (now.keys >> (kb * 16 + lane / 4 + (e >> 1) * 8)) & 1;
              float s = s2[kb][0][nt][e];
#pragma unroll
              for (int c = 1; c < CH; ++c) s += s2[kb][c][nt][e];
              p[kb][nt][e] = on ? s * a.scale : -INFINITY;
            }
            if (a.scores) {
              const int g = nt * 8 + lane % 4 * 2;
              float* to = a.scores + (((long long)now.row * a.kv.kv_heads + now.head) * a.mass_len + now.t * a.tile +
                                      warp * KEYS + kb * 16 + lane / 4) * a.group + now.g0 + g;
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if ((now.keys >> (kb * 16 + lane / 4 + (e >> 1) * 8)) & 1 && g + (e & 1) < live_g)
                  to[(e >> 1) * 8 * a.group + (e & 1)] = p[kb][nt][e];
            }
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float top = fmaxf(p[0][nt][e], p[0][nt][e + 2]);
#pragma unroll
            for (int kb = 1; kb < KB; ++kb) top = fmaxf(top, fmaxf(p[kb][nt][e], p[kb][nt][e + 2]));
#pragma unroll
            for (int x = 4; x < 32; x *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
            high[nt][e] = fmaxf(m[nt][e], top);
            moved |= high[nt][e] != m[nt][e];
          }
        }
        if (__any_sync(0xffffffffu, moved)) {  // a new maximum: rescale what is there
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float keep = exp2f(m[nt][e] - (high[nt][e] == -INFINITY ? 0.f : high[nt][e]));
              m[nt][e] = high[nt][e];
              l[nt][e] *= keep;
#pragma unroll
              for (int k = 0; k < MT; ++k) {
                o[k][nt][e] *= keep;
                o[k][nt][e + 2] *= keep;
              }
            }
        }
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float top = m[nt][e & 1];
              const bool on = (now.keys >> (kb * 16 + lane / 4 + (e >> 1) * 8)) & 1;
              p[kb][nt][e] = on ? exp2f(p[kb][nt][e] - (top == -INFINITY ? 0.f : top)) : 0.f;
              l[nt][e & 1] += p[kb][nt][e];
            }
        if constexpr (BF) {
          // parts of the weights, transposed; the last one is rounded, the least value
          // of bf16 in place of a zero part (an infinite value stays infinite)
          uint32_t b[KB][PS][NT][2];
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                float x = p[kb][nt][half * 2], y = p[kb][nt][half * 2 + 1];
                const bool xz = x == 0.f, yz = y == 0.f;
#pragma unroll
                for (int i = 0; i < PS - 1; ++i) b[kb][i][nt][half] = cut2(x, y);
                __nv_bfloat162 r = __floats2bfloat162_rn(x, y);
                b[kb][PS - 1][nt][half] = *reinterpret_cast<uint32_t*>(&r);
#pragma unroll
                for (int i = 0; i < PS; ++i) {
                  uint32_t& w = b[kb][i][nt][half];
                  if (i > 0 && !xz && !(w & 0xffffu)) w |= 1u;
                  if (i > 0 && !yz && !(w >> 16)) w |= 0x10000u;
                  w = transpose8(w);
                }
              }
#pragma unroll
          for (int k = 0; k < MT; ++k) {
            float x[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) x[nt][0] = x[nt][1] = x[nt][2] = x[nt][3] = 0.f;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
              uint32_t vf[4];
              ldsm_t(vf, vc + swz<C::kRow>(kb * 16 + (mi >> 1) * 8 + mr, k * 2 + (mi & 1)));
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = PS - 1; i >= 0; --i) mma(x[nt], vf, b[kb][i][nt][0], b[kb][i][nt][1]);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[k][nt][e] += x[nt][e];
          }
        } else {
          // weights of keys (2 t, 2 t + 1), t = lane % 4, of query lane / 4: two 16-bit
          // transposes each; the products' key order is the values' below
          float bh[2][NT][2], bl[2][NT][2];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const uint32_t x = __float_as_uint(p[0][nt][half * 2]), y = __float_as_uint(p[0][nt][half * 2 + 1]);
              const uint32_t low = transpose8(__byte_perm(x, y, 0x5410)), up = transpose8(__byte_perm(x, y, 0x7632));
              bl[half][nt][0] = __uint_as_float(__byte_perm(low, up, 0x5410));
              bl[half][nt][1] = __uint_as_float(__byte_perm(low, up, 0x7632));
#pragma unroll
              for (int e = 0; e < 2; ++e) {  // rounded, as the queries; a weight is 1 at the most
                float& w = bl[half][nt][e];
                bh[half][nt][e] = __uint_as_float(__float_as_uint(round_tf32(w)) & 0xffffe000u);
                w = w == w ? round_tf32(w - bh[half][nt][e]) : w;
              }
            }
          auto weigh = [&](int k) {
            float x[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) x[nt][0] = x[nt][1] = x[nt][2] = x[nt][3] = 0.f;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              // channel k 16 + lane / 4 (+ 8), keys half 8 + 2 (lane % 4) (+ 1): 32 different banks
              float lo[4], hi[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int r = half * 8 + lane % 4 * 2 + (e >> 1), c = k * 4 + (e & 1) * 2 + lane / 16;
                asm volatile("ld.shared.f32 %0, [%1];"
                             : "=f"(lo[e])
                             : "r"(vc + swz<C::kRow>(r, c) + lane / 4 % 4 * 4)
                             : "memory");
                hi[e] = cut_tf32(lo[e]);
              }
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma_tf32(x[nt], lo, bh[half][nt][0], bh[half][nt][1]);
                mma_tf32(x[nt], hi, bl[half][nt][0], bl[half][nt][1]);
                mma_tf32(x[nt], hi, bh[half][nt][0], bh[half][nt][1]);
              }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[k][nt][e] += x[nt][e];
          };
#pragma unroll
          for (int k = 0; k < MT1; ++k) weigh(k);
          if (MT1 < MT && d > DP1) {
#pragma unroll
            for (int k = MT1; k < MT; ++k) weigh(k);
          }
        }
      }
      __syncwarp();
    }
    if (walk.ahead > 0) {  // the stage's next chunk
      constexpr int SEGS = Walk<WHOLE, KEYS>::kSegs;
      long long off[SEGS];
      int no_page;
      const uint32_t keys = walk.chunk(a, off, &no_page);
      if (lane == 0) info[warp][st] = walk.info(a, keys, no_page, NT * 8);
      const uint32_t kd = smem_addr(ring + st * 2 * C::kChunkBytes), vd = kd + C::kChunkBytes;
#pragma unroll
      for (int i = 0; i < KEYS / KG; ++i) {
        const int r = i * KG + kg;  // KG divides 8: one eight for all lanes
        const bool on = (keys >> r) & 1;
        long long at;
        if (WHOLE)
          at = off[i * KG / kKvSegment] + (i * KG % kKvSegment + kg) * a.kv.slot_stride;
        else
          at = __shfl_sync(0xffffffffu, off[0], r);
        if (!on) at = 0;  // nothing is read
#pragma unroll
        for (int w = 0; w < CW; ++w) {
          const int cc = col + w * WIDE;
          if (cc < cols) {
            copy16(kd + swz<C::kRow>(r, cc), a.kv.k + at + cc * 16, on ? 16 : 0);
            copy16(vd + swz<C::kRow>(r, cc), a.kv.v + at + cc * 16, on ? 16 : 0);
          }
        }
      }
      walk.next(a);
    }
    copy_commit();
    st = st + 1 == S ? 0 : st + 1;
    if (!work) {
      ++filled;
      __syncwarp();
      continue;
    }
    --left;
    const int t = now.t, tiles = now.tiles, h = now.head, row = now.row, g0 = now.g0;
    if (t + 1 < tiles && left > 0) continue;
    // the unit ends here, or the CTA's part of it: the warps' pieces join
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int x = 4; x < 32; x *= 2) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], x);
        if (lane < 4) {
          float* to = ml + (warp * NT * 8 + nt * 8 + lane * 2 + e) * 2;
          to[0] = m[nt][e];
          to[1] = l[nt][e];
        }
      }
    if (bad && lane == 0) spoiled = 1;
    const bool whole = !CLUSTER && first_t == 0 && t + 1 == tiles;
    if (!CLUSTER && first_t == 0 && !whole && threadIdx.x == 0)  // begins here, ends behind
      a.cut[blockIdx.x] = CutUnit{row, h, g0, tiles, begin, run.total};
#pragma unroll 1
    for (int q4 = 0; q4 * kMergeHeads < live_g; ++q4) {
      if (lane % 4 / 2 == q4 % 2) {
        float* to = merge + (warp * kMergeHeads + lane % 2 * 2) * DP + lane / 4;
#pragma unroll
        for (int k = 0; k < MT; ++k) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            to[(e & 1) * DP + k * 16 + (e >> 1) * 8] = NT > 1 && q4 >= 2 ? o[k][NT - 1][e] : o[k][0][e];
        }
      }
      __syncthreads();
      const bool nan = spoiled != 0;
      if (nan && q4 == 0 && threadIdx.x == 0) kv_report(a.status, ER_KV_BAD_PAGE);
#pragma unroll 1
      for (int i = threadIdx.x; i < kMergeHeads * DP / 4; i += W * 32) {
        const int g4 = i / (DP / 4), cc = i % (DP / 4) * 4, g = q4 * kMergeHeads + g4;
        if (g >= live_g || cc >= d) continue;
        float2 p[W];
        float top = -INFINITY, sum = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < W; ++w) {
          p[w] = *reinterpret_cast<const float2*>(ml + (w * NT * 8 + g) * 2);
          top = fmaxf(top, p[w].x);
        }
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const float by = piece_weight(p[w].x, top);
          sum = fmaf(p[w].y, by, sum);
          fma4(acc, *reinterpret_cast<const float4*>(merge + (w * kMergeHeads + g4) * DP + cc), by);
        }
        if (nan) sum = __int_as_float(0x7fc00000);
        if (CLUSTER) {
          *reinterpret_cast<float4*>(piece_o + g * DP + cc) = acc;
          if (cc == 0) *reinterpret_cast<float2*>(piece_ml + g * 2) = make_float2(top, sum);
        } else if (whole) {
          const long long at = (long long)row * a.heads + h * a.group + g0 + g;
          kv_store4((TQ*)a.out + at * d + cc, acc, sum);
          if (a.scores && cc == 0) a.lse[at] = sum == 0.f ? INFINITY : top + log2f(sum);
        } else {
          const long long piece = ((long long)blockIdx.x * 2 + (first_t != 0 ? 0 : 1)) * (NT * 8) + g;
          *reinterpret_cast<float4*>(a.part_o + piece * d + cc) = acc;
          if (cc == 0) *reinterpret_cast<float2*>(a.part_ml + piece * 2) = make_float2(top, sum);
        }
      }
      __syncthreads();
    }
    if (left == 0) {
      if (CLUSTER) kv_cluster_join<TQ>(a, run, NT * 8, piece_ml, piece_o, DP);
      return;
    }
    fresh = true;
    begin += kv_cost(tiles);
  }
}

namespace {

template <typename TC, typename TQ, int DP, int NT, bool WHOLE, bool CLUSTER>
int attend_launch(const AttendArgs& a, cudaStream_t st) {
  using C = Mma<TC, TQ, DP, NT>;
  auto kernel = kv_attend_kernel<TC, TQ, DP, NT, WHOLE, CLUSTER>;
  static std::atomic<unsigned long long> done;
  if (int rc = allow_smem(kernel, C::kSmem, done)) return rc;
  return kv_launch(kernel, dim3(CLUSTER ? a.entries * a.units * kClusterCtas : a.grid), C::kWarps * 32, C::kSmem, CLUSTER,
                   st, "kv_attend_kernel", a);
}

template <typename TC, typename TQ, int DP, int NT>
int attend_go(const AttendArgs& a, cudaStream_t st) {
  if (a.kv.page_size % kKvSegment)
    return a.cluster ? attend_launch<TC, TQ, DP, NT, false, true>(a, st)
                     : attend_launch<TC, TQ, DP, NT, false, false>(a, st);
  return a.cluster ? attend_launch<TC, TQ, DP, NT, true, true>(a, st)
                   : attend_launch<TC, TQ, DP, NT, true, false>(a, st);
}

// Groups of more than 8 queries go 16 at a time, where the queries' parts
// leave room beside the ring.
template <typename TC>
bool attend_wide(int d, int group) { return group > 8 && !(sizeof(TC) == 4 && d > 128); }

template <typename TC, typename TQ>
int attend_dp(const AttendArgs& a, cudaStream_t st) {
  const bool wide = attend_wide<TC>(a.kv.d, a.group);
  if (a.kv.d <= 64) return wide ? attend_go<TC, TQ, 64, 2>(a, st) : attend_go<TC, TQ, 64, 1>(a, st);
  if (a.kv.d <= 128) return wide ? attend_go<TC, TQ, 128, 2>(a, st) : attend_go<TC, TQ, 128, 1>(a, st);
  if constexpr (sizeof(TC) == 2)
    if (wide) return attend_go<TC, TQ, 256, 2>(a, st);
  return attend_go<TC, TQ, 256, 1>(a, st);
}

template <typename TC, typename TQ, int DP, int NT>
KernelShape shape_of() {
  using C = Mma<TC, TQ, DP, NT>;
  return KernelShape{NT * 8, C::kWarps * C::kKeys, C::kSmem, C::kPerSm};
}
template <typename TC, typename TQ>
KernelShape shape_dp(int d, int group) {
  const bool wide = attend_wide<TC>(d, group);
  if (d <= 64) return wide ? shape_of<TC, TQ, 64, 2>() : shape_of<TC, TQ, 64, 1>();
  if (d <= 128) return wide ? shape_of<TC, TQ, 128, 2>() : shape_of<TC, TQ, 128, 1>();
  if constexpr (sizeof(TC) == 2)
    if (wide) return shape_of<TC, TQ, 256, 2>();
  return shape_of<TC, TQ, 256, 1>();
}

}  // namespace
}  // namespace er
