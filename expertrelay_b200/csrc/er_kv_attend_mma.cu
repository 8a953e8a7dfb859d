// er_kv_attend_mma.cu -- attention over a bf16 paged key-value cache on the
// tensor cores.
//
// One key and its value are 4 d bytes and take part in 4 d G flop, so the
// cache streams from memory while the arithmetic waits, as long as no lane
// touches each value G times: the products of a 16-key chunk with the
// group's queries run as m16n8k16 matrix instructions, keys (scores) or
// channels (values) along m and up to 8 queries along n, which pads a group
// of one to 8 columns for nothing but idle tensor cores. tcgen05 would take
// 64 rows of keys at the least, its operands and results through tensor
// memory; a chunk that one warp loads, multiplies and drops needs no
// barrier between warps at all.
//
//   scores^T [16 keys x 8 queries]  = K [16 x d] (ldmatrix) . Q^T (registers' order in shared memory)
//   out^T    [d x 8 queries]       += V^T [d x 16 keys] (ldmatrix.trans) . P^T [16 keys x 8 queries]
//
// The scores' accumulator turns into the second product's operand by two
// 8x8 transposes (movmatrix). bf16 has 8 bits, fp32 24: fp32 queries enter
// as the exact sum of three bf16 parts; the weights as two parts (16 bits,
// under a quarter of the rounding of a bf16 result) for bf16 results and as
// three (24 bits) for fp32 ones. Parts are cut, not rounded, so that they
// share the sign of the whole and an infinite key or value stays infinite.
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

constexpr int kMmaWarps = 4;
constexpr int kMergeHeads = 4;  // queries whose pieces the warps exchange at a time

template <int DP, int NT, int QS>
struct MmaRing {
  // about 96 KB a CTA (two fit an SM), 192 KB at DP = 256 (128 where the queries take 24)
  static constexpr int kStages = DP == 64 ? 6 : DP == 256 && NT * QS == 6 ? 2 : 3;
  static constexpr int kRow = DP * 2;               // bytes of a key in shared memory
  static constexpr int kChunkBytes = kKvChunk * kRow;
  static constexpr int kBytes = kMmaWarps * kStages * 2 * kChunkBytes;
};

template <int DP, int NT, int QS>
constexpr int mma_smem() {
  static_assert(MmaRing<DP, NT, QS>::kBytes + DP / 16 * QS * NT * 256 + 64 * DP + NT * 256 <= 228 * 1024 - 3072, "");
  return MmaRing<DP, NT, QS>::kBytes + DP / 16 * QS * NT * 32 * 8 + kMmaWarps * kMergeHeads * DP * 4 +
         kMmaWarps * NT * 8 * 2 * 4;
}

// Byte offset of the 16-byte column `col` of row `row`: columns permuted
// within each 128 bytes by the row, so that 8 rows' copies of one column lie
// in 8 different bank groups.
template <int DP>
__device__ __forceinline__ int swz(int row, int col) {
  return row * (DP * 2) + ((col ^ (row & 7)) << 4);
}

}  // namespace

// DP: head_dim padded to 64, 128 or 256; NT: tiles of 8 queries; QS: bf16
// parts of a query (1: bf16 queries and results, 3: fp32).
// WHOLE: page_size is a multiple of 16. CLUSTER: a cluster per unit.
template <int DP, int NT, int QS, bool WHOLE, bool CLUSTER>
__global__ void __launch_bounds__(kMmaWarps * 32, DP <= 128 && NT == 1 ? 2 : 1)
    kv_attend_mma_kernel(const __grid_constant__ AttendArgs a) {
  using Ring = MmaRing<DP, NT, QS>;
  constexpr int S = Ring::kStages, KS = DP / 16, PS = QS == 1 ? 2 : 3;
  extern __shared__ __align__(128) char sm[];
  __shared__ RunScratch scratch;
  __shared__ int spoiled;
  __shared__ StageInfo info[kMmaWarps][S];
  const int d = a.kv.d, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  char* ring = sm + warp * S * 2 * Ring::kChunkBytes;
  uint2* qf = reinterpret_cast<uint2*>(sm + Ring::kBytes);               // [KS][QS][NT][32]
  float* merge = reinterpret_cast<float*>(qf + KS * QS * NT * 32);       // [warps][kMergeHeads][DP]
  float* ml = merge + kMmaWarps * kMergeHeads * DP;                      // [warps][NT * 8][2]
  const int cols = d / 8;       // 16-byte columns of a row
  constexpr int W = DP / 8 < 32 ? DP / 8 : 32;  // lanes across a row
  const int col = lane % W, kg = lane / W;
  constexpr int KG = 32 / W;

  if (d < DP) {  // the columns behind head_dim stay zero
    for (int i = lane; i < S * 2 * kKvChunk * (DP / 8); i += 32)
      *reinterpret_cast<uint4*>(ring + i * 16) = make_uint4(0, 0, 0, 0);
    __syncwarp();
  }
  kv_enter();
  using TQ = std::conditional_t<QS == 1, __nv_bfloat16, float>;
  // a cluster's CTA leaves its piece where its ring was
  float *piece_ml = reinterpret_cast<float*>(sm), *piece_o = piece_ml + NT * 8 * 2;
  const Run run = CLUSTER ? kv_cluster_run(a) : kv_run(a, scratch);
  if (run.left == 0) {
    if (CLUSTER) {
      __syncthreads();  // the ring's zeros are written
      for (int i = threadIdx.x; i < NT * 8 * (DP + 2); i += kMmaWarps * 32)
        piece_ml[i] = i < NT * 16 && !(i & 1) ? -INFINITY : 0.f;
      kv_cluster_join<TQ>(a, run, NT * 8, piece_ml, piece_o, DP);
    }
    return;
  }
  long long left = run.left, begin = run.begin;
  Walk<WHOLE> walk(a, run);

  float m[NT][2], l[NT][2], o[KS][NT][4];
  bool fresh = true, bad = false;
  int st = 0, first_t = 0, live_g = 0, filled = 0;
  // One loop fills the ring (S steps), then takes a stage and fills it again:
  // each piece of code stands once, since a short launch waits for its
  // instructions as it does for its data.
#pragma unroll 1
  for (;;) {
    const bool work = filled == S;
    StageInfo now = {};
    if (work) now = info[warp][st];
    // a new unit: its queries in the matrix instructions' order (the first
    // unit's before the ring is filled, while its pages are looked up)
    if (fresh && (work || filled == 0)) {
      if (!work) now = walk.info(a, 0, NT * 8);
      fresh = false;
      bad = false;
      first_t = now.t;
      live_g = min(NT * 8, a.group - now.g0);
      const long long qat = (long long)now.row * a.q_stride + (long long)(now.head * a.group + now.g0) * d;
#pragma unroll 2
      for (int i = threadIdx.x; i < KS * NT * 32; i += kMmaWarps * 32) {
        const int ln = i % 32, nt = i / 32 % NT, ks = i / (32 * NT);
        const int g = nt * 8 + ln / 4, c0 = ks * 16 + ln % 4 * 2;
        if constexpr (QS == 1) {
          uint32_t x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int cc = c0 + (e & 1) + (e >> 1) * 8;
            x[e] = g < live_g && cc < d ? (uint32_t)reinterpret_cast<const uint16_t*>(a.q)[qat + (long long)g * d + cc] : 0u;
          }
          qf[i] = make_uint2(x[0] | x[1] << 16, x[2] | x[3] << 16);
        } else {
          float x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int cc = c0 + (e & 1) + (e >> 1) * 8;
            x[e] = g < live_g && cc < d ? reinterpret_cast<const float*>(a.q)[qat + (long long)g * d + cc] : 0.f;
          }
          uint32_t p[4][QS];
#pragma unroll
          for (int e = 0; e < 4; ++e) query_parts(x[e], p[e]);
#pragma unroll
          for (int part = 0; part < QS; ++part)
            qf[((ks * QS + part) * NT + nt) * 32 + ln] =
                make_uint2(p[0][part] | p[1][part] << 16, p[2][part] | p[3][part] << 16);
        }
      }
      if (threadIdx.x == 0) spoiled = 0;
      __syncthreads();
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        m[nt][0] = m[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
        for (int k = 0; k < KS; ++k) o[k][nt][0] = o[k][nt][1] = o[k][nt][2] = o[k][nt][3] = 0.f;
      }
    }
    if (work) {
    copy_wait<S - 1>();
    __syncwarp();
    const uint32_t mask = now.keys;
    if (mask >> 16) bad = true;
    if (mask & 0xffff) {
      const uint32_t kc = smem_addr(ring + st * 2 * Ring::kChunkBytes), vc = kc + Ring::kChunkBytes;
      const int mi = lane / 8, mr = lane % 8;  // the 8x8 matrix and its row that this lane addresses
      // two chains of products: their latencies overlap, and each is summed
      // over half as many steps (the parts below the leading one in the second)
      float s2[2][NT][4];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s2[i][nt][0] = s2[i][nt][1] = s2[i][nt][2] = s2[i][nt][3] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        uint32_t kf[4];
        ldsm(kf, kc + swz<DP>((mi & 1) * 8 + mr, ks * 2 + (mi >> 1)));
#pragma unroll
        for (int p = 0; p < QS; ++p)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const uint2 b = qf[((ks * QS + p) * NT + nt) * 32 + lane];
            mma(s2[QS == 1 ? ks & 1 : p > 0][nt], kf, b.x, b.y);
          }
      }
      const bool on0 = (mask >> (lane / 4)) & 1, on1 = (mask >> (lane / 4 + 8)) & 1;
      float high[NT][2], p[NT][4];
      bool moved = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float(&s)[4] = p[nt];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[e] = (s2[0][nt][e] + s2[1][nt][e]) * a.scale;
          if (!(e < 2 ? on0 : on1)) s[e] = -INFINITY;
        }
        if (a.scores) {
          const int g = nt * 8 + lane % 4 * 2;
          float* to = a.scores + (((long long)now.row * a.kv.kv_heads + now.head) * a.mass_len + now.t * a.tile +
                                  warp * kKvChunk + lane / 4) * a.group + now.g0 + g;
          if (on0 && g < live_g) to[0] = s[0];
          if (on0 && g + 1 < live_g) to[1] = s[1];
          to += 8 * a.group;
          if (on1 && g < live_g) to[0] = s[2];
          if (on1 && g + 1 < live_g) to[1] = s[3];
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = fmaxf(s[e], s[e + 2]);
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
            for (int k = 0; k < KS; ++k) {
              o[k][nt][e] *= keep;
              o[k][nt][e + 2] *= keep;
            }
          }
      }
      uint32_t b[PS][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float top = m[nt][e & 1];
          p[nt][e] = (e < 2 ? on0 : on1) ? exp2f(p[nt][e] - (top == -INFINITY ? 0.f : top)) : 0.f;
          l[nt][e & 1] += p[nt][e];
        }
        // parts of the weights; the last one is rounded, the least value of
        // bf16 in place of a zero part (an infinite value stays infinite)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float x = p[nt][half * 2], y = p[nt][half * 2 + 1];
          const bool xz = x == 0.f, yz = y == 0.f;
#pragma unroll
          for (int i = 0; i < PS - 1; ++i) b[i][nt][half] = cut2(x, y);
          __nv_bfloat162 r = __floats2bfloat162_rn(x, y);
          b[PS - 1][nt][half] = *reinterpret_cast<uint32_t*>(&r);
#pragma unroll
          for (int i = 1; i < PS; ++i) {
            if (!xz && !(b[i][nt][half] & 0xffffu)) b[i][nt][half] |= 1u;
            if (!yz && !(b[i][nt][half] >> 16)) b[i][nt][half] |= 0x10000u;
          }
#pragma unroll
          for (int i = 0; i < PS; ++i) b[i][nt][half] = transpose8(b[i][nt][half]);
        }
      }
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        uint32_t vf[4];
        ldsm_t(vf, vc + swz<DP>((mi >> 1) * 8 + mr, k * 2 + (mi & 1)));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if (QS == 1) {
#pragma unroll
            for (int i = PS - 1; i >= 0; --i) mma(o[k][nt], vf, b[i][nt][0], b[i][nt][1]);
          } else {  // the tensor cores cut their sums: a chunk's alone there, the running sum rounded here
            float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = PS - 1; i >= 0; --i) mma(x, vf, b[i][nt][0], b[i][nt][1]);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[k][nt][e] += x[e];
          }
        }
      }
    }
    __syncwarp();
    }
    if (walk.ahead > 0) {  // the stage's next chunk
      long long off = 0;
      const uint32_t keys = walk.chunk(a, &off);
      if (lane == 0) info[warp][st] = walk.info(a, keys, NT * 8);
      const uint32_t kd = smem_addr(ring + st * 2 * Ring::kChunkBytes), vd = kd + Ring::kChunkBytes;
      if (col < cols || !WHOLE) {
        const long long step = kg * a.kv.slot_stride + col * 16;
        const char *kp = a.kv.k + off + step, *vp = a.kv.v + off + step;
#pragma unroll
        for (int i = 0; i < kKvChunk / KG; ++i) {
          const int r = i * KG + kg, bytes = (keys >> r) & 1 ? 16 : 0;
          if (!WHOLE) {
            const long long at = __shfl_sync(0xffffffffu, off, r);
            kp = a.kv.k + (at >= 0 ? at : 0) + col * 16;
            vp = a.kv.v + (at >= 0 ? at : 0) + col * 16;
          }
          if (WHOLE || col < cols) {
            // a key that is not there is not read: its address is the pool's first
            copy16(kd + swz<DP>(r, col), bytes ? kp : a.kv.k, bytes);
            copy16(vd + swz<DP>(r, col), bytes ? vp : a.kv.v, bytes);
          }
          kp += KG * a.kv.slot_stride;
          vp += KG * a.kv.slot_stride;
        }
      }
      walk.next(a);
    }
    copy_commit();
    st = st + 1 == S ? 0 : st + 1;
    if (!work) {
      ++filled;
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
        for (int k = 0; k < KS; ++k) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            to[(e & 1) * DP + k * 16 + (e >> 1) * 8] = NT > 1 && q4 >= 2 ? o[k][NT - 1][e] : o[k][0][e];
        }
      }
      __syncthreads();
      const bool nan = spoiled != 0;
      if (nan && q4 == 0 && threadIdx.x == 0) kv_report(a.status, ER_KV_BAD_PAGE);
#pragma unroll 1
      for (int i = threadIdx.x; i < kMergeHeads * DP / 4; i += kMmaWarps * 32) {
        const int g4 = i / (DP / 4), cc = i % (DP / 4) * 4, g = q4 * kMergeHeads + g4;
        if (g >= live_g || cc >= d) continue;
        float2 p[kMmaWarps];
        float top = -INFINITY, sum = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kMmaWarps; ++w) {
          p[w] = *reinterpret_cast<const float2*>(ml + (w * NT * 8 + g) * 2);
          top = fmaxf(top, p[w].x);
        }
#pragma unroll
        for (int w = 0; w < kMmaWarps; ++w) {
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

template <int DP, int NT, int QS, bool WHOLE, bool CLUSTER>
int mma_launch(const AttendArgs& a, cudaStream_t st) {
  auto kernel = kv_attend_mma_kernel<DP, NT, QS, WHOLE, CLUSTER>;
  constexpr int smem = mma_smem<DP, NT, QS>();
  static_assert(NT * 8 * (DP + 2) * 4 <= MmaRing<DP, NT, QS>::kBytes, "a piece fits the ring");
  static std::atomic<unsigned long long> done;
  if (int rc = allow_smem(kernel, smem, done)) return rc;
  return kv_launch(kernel, dim3(CLUSTER ? a.entries * a.units * kClusterCtas : a.grid), kMmaWarps * 32, smem, CLUSTER, st,
                   "kv_attend_mma_kernel", a);
}

template <int DP, int NT, int QS>
int mma_go(const AttendArgs& a, cudaStream_t st) {
  if (a.kv.page_size % kKvChunk)
    return a.cluster ? mma_launch<DP, NT, QS, false, true>(a, st) : mma_launch<DP, NT, QS, false, false>(a, st);
  return a.cluster ? mma_launch<DP, NT, QS, true, true>(a, st) : mma_launch<DP, NT, QS, true, false>(a, st);
}

template <int NT, int QS>
int mma_dp(const AttendArgs& a, cudaStream_t st) {
  if (a.kv.d <= 64) return mma_go<64, NT, QS>(a, st);
  if (a.kv.d <= 128) return mma_go<128, NT, QS>(a, st);
  return mma_go<256, NT, QS>(a, st);
}

template <int NT, int QS>
int smem_dp(int d) {
  return d <= 64 ? mma_smem<64, NT, QS>() : d <= 128 ? mma_smem<128, NT, QS>() : mma_smem<256, NT, QS>();
}

}  // namespace

KernelShape mma_shape(int d, int group, int q_dtype) {
  KernelShape s;
  const int nt = group > 8 ? 2 : 1;
  s.heads = nt * 8;
  s.warps = kMmaWarps;
  s.smem = q_dtype == ER_DTYPE_BF16 ? (nt == 1 ? smem_dp<1, 1>(d) : smem_dp<2, 1>(d))
                                    : (nt == 1 ? smem_dp<1, 3>(d) : smem_dp<2, 3>(d));
  s.per_sm = nt == 1 && 2 * (s.smem + 3072) <= 227 * 1024 ? 2 : 1;
  return s;
}

int attend_mma(const AttendArgs& a, int q_dtype, cudaStream_t st) {
  const int nt = a.group > 8 ? 2 : 1;
  if (q_dtype == ER_DTYPE_BF16) return nt == 1 ? mma_dp<1, 1>(a, st) : mma_dp<2, 1>(a, st);
  return nt == 1 ? mma_dp<1, 3>(a, st) : mma_dp<2, 3>(a, st);
}

}  // namespace er
