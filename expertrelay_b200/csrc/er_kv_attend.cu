// er_kv_attend.cu -- attention of rows of queries over the paged key-value
// cache: the fp32 kernel, the join of split rows, the accumulated attention
// weight, and the entry point.
#include "er_kv_attend.cuh"

namespace er {

constexpr int kSimtStages = 3;

// Shared memory of the fp32 kernel: queries, the warps' pieces, probabilities,
// then per warp a ring of kSimtStages chunks of keys and values, their rows
// an odd number of 16-byte columns apart (no bank conflicts across keys).
inline int simt_pitch(int d) { return d * 4 + ((d / 4) % 2 ? 0 : 16); }
// `most`: 220 KB for one CTA an SM, half of it for two.
inline KernelShape simt_shape(int d, int group, int most) {
  KernelShape s;
  s.heads = group <= 1 ? 1 : group <= 2 ? 2 : group <= 4 ? 4 : 8;
  for (s.warps = 4; s.warps > 1; s.warps /= 2) {
    s.smem = s.heads * d * 4 + s.warps * s.heads * (d + 4) * 4 + s.warps * s.heads * kKvChunk * 4 + 64 +
             s.warps * kSimtStages * (2 * kKvChunk * simt_pitch(d));
    if (s.smem <= most) break;
  }
  s.per_sm = 227 * 1024 / (s.smem + 3072);
  if (s.per_sm > 4) s.per_sm = 4;
  return s;
}

// fp32 throughout: a warp takes 16 keys at a time, from its own ring of
// asynchronous copies. Scores: lane l holds key l % 16 and half of the
// columns. Values: the lanes split a row's 16-byte columns, lane groups the
// keys. GB queries of the group at a time share each key that is read.
template <typename TQ, int GB, bool WHOLE, bool CLUSTER>
__global__ void __launch_bounds__(128) kv_attend_simt_kernel(const __grid_constant__ AttendArgs a, int pitch) {
  using TC = float;
  constexpr int V = 16 / sizeof(TC);
  extern __shared__ __align__(16) char sm[];
  __shared__ RunScratch scratch;
  __shared__ int spoiled;
  __shared__ StageInfo info[4][kSimtStages];
  const int d = a.kv.d, warps = blockDim.x / 32, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float* qs = reinterpret_cast<float*>(sm);                // [GB][d]
  const int pitch_m = d + 4;
  float* merge = qs + GB * d;                              // [warps][GB][d + 4]: o, m, l
  float* prob = merge + warps * GB * pitch_m + warp * GB * kKvChunk;  // [16][GB]
  char* ring0 = sm + (GB * d + warps * GB * pitch_m + warps * GB * kKvChunk) * 4;
  char* ring = ring0 + warp * kSimtStages * 2 * kKvChunk * pitch;
  const int cols = d / V;
  int wide = 2;  // lanes across a row; at most 16 rows at a time, so every lane group has as many
  while (wide < cols && wide < 32) wide *= 2;
  const int col = lane % wide, kg = lane / wide, kgs = 32 / wide;

  kv_enter();
  // a cluster's CTA leaves its piece where its ring was
  float *piece_ml = reinterpret_cast<float*>(ring0), *piece_o = piece_ml + (GB * 2 + 3) / 4 * 4;
  const Run run = CLUSTER ? kv_cluster_run(a) : kv_run(a, scratch);
  if (run.left == 0) {
    if (CLUSTER) {
      for (int i = threadIdx.x; i < GB * 2; i += blockDim.x) piece_ml[i] = i & 1 ? 0.f : -INFINITY;
      for (int i = threadIdx.x; i < GB * d; i += blockDim.x) piece_o[i] = 0.f;
      kv_cluster_join<TQ>(a, run, GB, piece_ml, piece_o, d);
    }
    return;
  }
  long long left = run.left, begin = run.begin;
  Walk<WHOLE> walk(a, run);

  float m[GB], l[GB], o[GB][8];
  bool fresh = true, bad = false;
  int st = 0, first_t = 0, filled = 0, live_g = 0;
  // One loop fills the ring, then takes a stage and fills it again: each
  // piece of code stands once, since a short launch waits for its
  // instructions as it does for its data.
#pragma unroll 1
  for (;;) {
    const bool work = filled == kSimtStages;
    StageInfo now = {};
    if (work) now = info[warp][st];
    // a new unit: its queries (the first unit's before the ring is filled,
    // while its pages are looked up)
    if (fresh && (work || filled == 0)) {
      if (!work) now = walk.info(a, 0, GB);
      fresh = false;
      bad = false;
      first_t = now.t;
      live_g = min(GB, a.group - now.g0);
      const TQ* q = (const TQ*)a.q + (long long)now.row * a.q_stride + (long long)(now.head * a.group + now.g0) * d;
      for (int i = threadIdx.x; i < GB * d; i += blockDim.x) qs[i] = i < live_g * d ? to_f32(q[i]) : 0.f;
      if (threadIdx.x == 0) spoiled = 0;
      __syncthreads();
#pragma unroll
      for (int g = 0; g < GB; ++g) {
        m[g] = -INFINITY;
        l[g] = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[g][e] = 0.f;
      }
    }
    if (work) {
    copy_wait<kSimtStages - 1>();
    __syncwarp();
    const uint32_t mask = now.keys;
    if (mask >> 16) bad = true;
    if (mask & 0xffff) {
      const char* kc = ring + st * 2 * kKvChunk * pitch;
      const char* vc = kc + kKvChunk * pitch;
      const int key = lane & 15;
      const bool on = (mask >> key) & 1;
      float s[GB];
#pragma unroll
      for (int g = 0; g < GB; ++g) s[g] = 0.f;
#pragma unroll 4
      for (int cc = lane >> 4; cc < cols; cc += 2) {
        const uint4 raw = *reinterpret_cast<const uint4*>(kc + key * pitch + cc * 16);
        const TC* kx = reinterpret_cast<const TC*>(&raw);
        float kf[V];
#pragma unroll
        for (int e = 0; e < V; ++e) kf[e] = to_f32(kx[e]);
#pragma unroll
        for (int g = 0; g < GB; ++g)
#pragma unroll
          for (int e = 0; e < V; e += 4) {
            const float4 qv = *reinterpret_cast<const float4*>(qs + g * d + cc * V + e);
            s[g] = fmaf(qv.x, kf[e], fmaf(qv.y, kf[e + 1], fmaf(qv.z, kf[e + 2], fmaf(qv.w, kf[e + 3], s[g]))));
          }
      }
#pragma unroll
      for (int g = 0; g < GB; ++g) {
        s[g] = (s[g] + __shfl_xor_sync(0xffffffffu, s[g], 16)) * a.scale;
        if (!on) s[g] = -INFINITY;
      }
      if (a.scores && on && lane < 16) {
        float* to = a.scores + (((long long)now.row * a.kv.kv_heads + now.head) * a.mass_len + now.t * a.tile +
                                warp * kKvChunk + key) * a.group + now.g0;
#pragma unroll
        for (int g = 0; g < GB; ++g)
          if (g < live_g) to[g] = s[g];
      }
#pragma unroll
      for (int g = 0; g < GB; ++g) {
        float top = s[g];
#pragma unroll
        for (int x = 8; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        const float high = fmaxf(m[g], top);
        const float base = high == -INFINITY ? 0.f : high;  // scores of -inf alone weigh nothing
        const float keep = exp2f(m[g] - base);
        m[g] = high;
        const float p = on ? exp2f(s[g] - base) : 0.f;
        l[g] = l[g] * keep + (lane < 16 ? p : 0.f);
        if (lane < 16) prob[key * GB + g] = p;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[g][e] *= keep;
      }
      __syncwarp();
#pragma unroll 4
      for (int r = kg; r < kKvChunk; r += kgs) {
        float p[GB];
#pragma unroll
        for (int g = 0; g < GB; ++g) p[g] = prob[r * GB + g];
#pragma unroll
        for (int w = 0; w < 8 / V; ++w) {
          const int cc = col + 32 * w;
          if (cc < cols) {
            const uint4 raw = *reinterpret_cast<const uint4*>(vc + r * pitch + cc * 16);
            const TC* vx = reinterpret_cast<const TC*>(&raw);
#pragma unroll
            for (int e = 0; e < V; ++e) {
              const float f = to_f32(vx[e]);
#pragma unroll
              for (int g = 0; g < GB; ++g) o[g][w * V + e] = fmaf(p[g], f, o[g][w * V + e]);
            }
          }
        }
      }
    }
    __syncwarp();
    }
    if (walk.ahead > 0) {  // the stage's next chunk
      long long off = 0;
      const uint32_t keys = walk.chunk(a, &off);
      if (lane == 0) info[warp][st] = walk.info(a, keys, GB);
      const uint32_t kd = smem_addr(ring + st * 2 * kKvChunk * pitch), vd = kd + kKvChunk * pitch;
#pragma unroll 4
      for (int r = kg; r < kKvChunk; r += kgs) {
        const long long at = WHOLE ? off + r * a.kv.slot_stride : __shfl_sync(0xffffffffu, off, r);
        const int bytes = (keys >> r) & 1 ? 16 : 0;
        // a key that is not there is not read: its address is the pool's first
        const char *kp = a.kv.k + (bytes ? at : 0), *vp = a.kv.v + (bytes ? at : 0);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const int cc = col + 32 * w;
          if (cc < cols) {
            copy16(kd + r * pitch + cc * 16, kp + (bytes ? cc * 16 : 0), bytes);
            copy16(vd + r * pitch + cc * 16, vp + (bytes ? cc * 16 : 0), bytes);
          }
        }
      }
      walk.next(a);
    }
    copy_commit();
    st = st + 1 == kSimtStages ? 0 : st + 1;
    if (!work) {
      ++filled;
      continue;
    }
    --left;
    const int t = now.t, tiles = now.tiles, h = now.head, row = now.row, g0 = now.g0;
    if (t + 1 < tiles && left > 0) continue;
    // the unit ends here, or the CTA's part of it: the warps' pieces join
#pragma unroll
    for (int g = 0; g < GB; ++g) {
      l[g] = warp_sum(l[g]);
#pragma unroll 1
      for (int x = wide; x < 32; x *= 2)
#pragma unroll
        for (int e = 0; e < 8; ++e) o[g][e] += __shfl_xor_sync(0xffffffffu, o[g][e], x);
      float* to = merge + (warp * GB + g) * pitch_m;
      if (lane == 0) {
        to[d] = m[g];
        to[d + 1] = l[g];
      }
      if (kg == 0) {
#pragma unroll
        for (int w = 0; w < 8 / V; ++w)
          if (col + 32 * w < cols) {
#pragma unroll
            for (int e = 0; e < V; ++e) to[(col + 32 * w) * V + e] = o[g][w * V + e];
          }
      }
    }
    if (bad && lane == 0) spoiled = 1;
    __syncthreads();
    const bool whole = !CLUSTER && first_t == 0 && t + 1 == tiles;
    if (!CLUSTER && first_t == 0 && !whole && threadIdx.x == 0)  // begins here, ends behind
      a.cut[blockIdx.x] = CutUnit{row, h, g0, tiles, begin, run.total};
    const bool nan = spoiled != 0;
    if (nan && threadIdx.x == 0) kv_report(a.status, ER_KV_BAD_PAGE);
#pragma unroll 1
    for (int i = threadIdx.x; i < live_g * cols; i += blockDim.x) {
      const int g = i / cols, cc = (i - g * cols) * 4;
      const float* from = merge + g * pitch_m;
      float top = -INFINITY, sum = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int w = 0; w < warps; ++w) top = fmaxf(top, from[w * GB * pitch_m + d]);
#pragma unroll 4
      for (int w = 0; w < warps; ++w) {
        const float* p = from + w * GB * pitch_m;
        const float by = piece_weight(p[d], top);
        sum = fmaf(p[d + 1], by, sum);
        fma4(acc, *reinterpret_cast<const float4*>(p + cc), by);
      }
      if (nan) sum = __int_as_float(0x7fc00000);
      if (CLUSTER) {
        *reinterpret_cast<float4*>(piece_o + g * d + cc) = acc;
        if (cc == 0) *reinterpret_cast<float2*>(piece_ml + g * 2) = make_float2(top, sum);
      } else if (whole) {
        const long long at = (long long)row * a.heads + h * a.group + g0 + g;
        kv_store4((TQ*)a.out + at * d + cc, acc, sum);
        if (a.scores && cc == 0) a.lse[at] = sum == 0.f ? INFINITY : top + log2f(sum);
      } else {
        const long long piece = ((long long)blockIdx.x * 2 + (first_t != 0 ? 0 : 1)) * GB + g;
        *reinterpret_cast<float4*>(a.part_o + piece * d + cc) = acc;
        if (cc == 0) *reinterpret_cast<float2*>(a.part_ml + piece * 2) = make_float2(top, sum);
      }
    }
    __syncthreads();
    if (left == 0) {
      if (CLUSTER) kv_cluster_join<TQ>(a, run, GB, piece_ml, piece_o, d);
      return;
    }
    fresh = true;
    begin += kv_cost(tiles);
  }
}

// Joins the units that several CTAs share: CTA (i, g) query g of the unit
// that begins in CTA i's run and ends behind it. The pieces are that CTA's
// last one and the first ones of the CTAs after it. A piece's weights are
// found once, then threads split the pieces and the channels (four each).
// The CTAs of g = 0 also write the rows without keys (zeros) and the bad
// ones (NaN), which no attention CTA meets.
constexpr int kJoinThreads = 256, kJoinPieces = 3;  // 768 pieces

template <typename TQ>
__global__ void __launch_bounds__(kJoinThreads) kv_join_kernel(const __grid_constant__ AttendArgs a, int gb) {
  extern __shared__ float wt[];  // [grid] weights, then [kJoinThreads][4] partial sums
  __shared__ float red[2][kJoinThreads / 32];
  kv_enter();
  const int g = blockIdx.y, d = a.kv.d;
  if (g == 0) {
    for (int x = blockIdx.x; x < a.entries; x += a.grid) {
      const Entry e = kv_entry(a, x);
      if (e.n > 0) continue;
      const TQ v = kv_round<TQ>(e.bad ? __int_as_float(0x7fc00000) : 0.f);
      const int per = (a.pages ? a.group : a.heads) * d;  // an entry is a row, or a key head of one
      TQ* out = (TQ*)a.out + (long long)x * per;
      for (int i = threadIdx.x; i < per; i += kJoinThreads) out[i] = v;
    }
  }
  const CutUnit c = a.cut[blockIdx.x];
  if (c.row < 0 || c.g0 + g >= a.group) return;
  const int shares = kv_shares(a, c.total), i0 = blockIdx.x;
  const int n = kv_share_of(c.total, shares, c.begin + kUnitCost + c.tiles - 1) - i0 + 1;  // pieces
  auto piece = [&](int k) { return ((long long)(i0 + k) * 2 + (k == 0 ? 1 : 0)) * gb + g; };
  // a thread has pieces tid, tid + 256 and tid + 512 (CTAs, so pieces, are 4 an SM at the most)
  float2 ml[kJoinPieces];
  float top = -INFINITY, sum = 0.f;
#pragma unroll
  for (int j = 0; j < kJoinPieces; ++j) {
    const int k = threadIdx.x + j * kJoinThreads;
    ml[j] = k < n ? *reinterpret_cast<const float2*>(a.part_ml + piece(k) * 2) : make_float2(-INFINITY, 0.f);
    top = fmaxf(top, ml[j].x);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (threadIdx.x % 32 == 0) red[0][threadIdx.x / 32] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kJoinThreads / 32; ++w) top = fmaxf(top, red[0][w]);
#pragma unroll
  for (int j = 0; j < kJoinPieces; ++j) {
    const int k = threadIdx.x + j * kJoinThreads;
    if (k < n) {
      wt[k] = piece_weight(ml[j].x, top);
      sum = fmaf(ml[j].y, wt[k], sum);  // a spoiled piece's sum is NaN
    }
  }
  sum = warp_sum(sum);
  if (threadIdx.x % 32 == 0) red[1][threadIdx.x / 32] = sum;
  __syncthreads();
  sum = 0.f;
#pragma unroll
  for (int w = 0; w < kJoinThreads / 32; ++w) sum += red[1][w];
  const int cols = d / 4, groups = kJoinThreads / cols;  // 2 .. 64 columns of 4 channels
  const int col = threadIdx.x % cols, grp = threadIdx.x / cols;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (grp < groups) {
#pragma unroll 8
    for (int k = grp; k < n; k += groups) {
      const float4 x = *reinterpret_cast<const float4*>(a.part_o + piece(k) * d + col * 4);
      const float by = wt[k];
      fma4(acc, x, by);
    }
  }
  float4* part = reinterpret_cast<float4*>(wt + (a.grid + 3) / 4 * 4);
  part[threadIdx.x] = acc;
  __syncthreads();
  const long long at = (long long)c.row * a.heads + c.head * a.group + c.g0 + g;
  if (threadIdx.x < cols) {
    for (int q = 1; q < groups; ++q) {
      const float4 x = part[q * cols + col];
      acc.x += x.x;
      acc.y += x.y;
      acc.z += x.z;
      acc.w += x.w;
    }
    kv_store4((TQ*)a.out + at * d + col * 4, acc, sum);
  }
  if (a.scores && threadIdx.x == 0) a.lse[at] = sum == 0.f ? INFINITY : top + log2f(sum);
}

// mass[row, h, j] += sum_g 2^(s_gj - lse_g), a thread per position.
__global__ void __launch_bounds__(256) kv_mass_kernel(const __grid_constant__ AttendArgs a) {
  kv_enter();
  const int unit = blockIdx.y, row = unit / a.kv.kv_heads, h = unit % a.kv.kv_heads;
  const Entry e = kv_entry(a, row);
  float* to = a.mass + row * a.mass_row_stride + h * a.mass_head_stride;
  const float* s = a.scores + (long long)unit * a.mass_len * a.group;
  const float* lse = a.lse + (long long)row * a.heads + h * a.group;
  for (int j = blockIdx.x * 256 + threadIdx.x; j < e.n; j += gridDim.x * 256) {
    float sum = 0.f;
    for (int g = 0; g < a.group; ++g) sum += exp2f(s[(long long)j * a.group + g] - lse[g]);
    to[j] += sum;
  }
}

namespace {

template <typename TQ, int GB, bool WHOLE, bool CLUSTER>
int simt_launch(const AttendArgs& a, const KernelShape& s, cudaStream_t st) {
  auto kernel = kv_attend_simt_kernel<TQ, GB, WHOLE, CLUSTER>;
  static std::atomic<unsigned long long> done;
  if (int rc = allow_smem(kernel, 224 * 1024, done)) return rc;
  return kv_launch(kernel, dim3(CLUSTER ? a.entries * a.units * kClusterCtas : a.grid), s.warps * 32, s.smem, CLUSTER, st,
                   "kv_attend_simt_kernel", a, simt_pitch(a.kv.d));
}

template <typename TQ, int GB>
int simt_go(const AttendArgs& a, const KernelShape& s, cudaStream_t st) {
  if (a.kv.page_size % kKvChunk)
    return a.cluster ? simt_launch<TQ, GB, false, true>(a, s, st) : simt_launch<TQ, GB, false, false>(a, s, st);
  return a.cluster ? simt_launch<TQ, GB, true, true>(a, s, st) : simt_launch<TQ, GB, true, false>(a, s, st);
}

template <typename TQ>
int attend_simt(const AttendArgs& a, const KernelShape& s, cudaStream_t st) {
  switch (s.heads) {
    case 1: return simt_go<TQ, 1>(a, s, st);
    case 2: return simt_go<TQ, 2>(a, s, st);
    case 4: return simt_go<TQ, 4>(a, s, st);
    default: return simt_go<TQ, 8>(a, s, st);
  }
}

constexpr int kMaxEntries = 4096;  // scan entries a launch takes; more rows go in several launches

struct Layout {
  KernelShape shape;
  int blocks, grid, rows;  // rows: of one launch
  bool cluster;
  size_t cut, ml, o, lse, scores, bytes;
};

Layout attend_layout(const er_kv_cache& c, const er_kv_attend_io& io, int sms) {
  Layout L;
  const int group = io.heads / c.kv_heads;
  const bool mma = c.dtype == ER_DTYPE_BF16;
  L.shape = mma ? mma_shape(c.head_dim, group, io.q_dtype) : simt_shape(c.head_dim, group, 220 * 1024);
  L.blocks = (group + L.shape.heads - 1) / L.shape.heads;
  L.grid = sms * L.shape.per_sm;
  if (L.grid > kJoinThreads * kJoinPieces) L.grid = kJoinThreads * kJoinPieces;
  L.rows = io.pages ? kMaxEntries / c.kv_heads : kMaxEntries;
  if (L.rows < 1) L.rows = 1;
  if (L.rows > io.rows) L.rows = io.rows;
  // A cluster per unit or equal shares of all tiles. Against the shares the
  // clusters save about 7 tiles' time (no division of the line, no join), but
  // a unit has 8 CTAs at most: taken while its longest row costs those CTAs
  // less than 7 tiles more than a share would be, and all clusters run at
  // once. That takes two CTAs an SM: with one, 16 clusters of 8 did not all
  // find room in the processor clusters of 148 SMs, and 16 units of 640
  // fp32 keys took 20 us, a wave after the other (14 by shares).
  const KernelShape half = mma ? L.shape : simt_shape(c.head_dim, group, 108 * 1024);
  const long long units = (long long)L.rows * c.kv_heads * L.blocks, tile = half.warps * kKvChunk, ctas = sms * 2;
  const long long longest =
      ((io.pages ? (long long)io.max_pages : (long long)c.table_width) * c.page_size + tile - 1) / tile;
  L.cluster = L.rows == io.rows && half.per_sm >= 2 && units * kClusterCtas <= ctas &&
              longest * (ctas - units * kClusterCtas) <= 7LL * kClusterCtas * ctas;
  if (L.cluster) L.shape = half;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += align_up(bytes, 256);
    return here;
  };
  const size_t pieces = L.cluster ? 0 : (size_t)L.grid * 2 * L.shape.heads;  // two a CTA
  L.cut = take(L.cluster ? 0 : (size_t)L.grid * sizeof(CutUnit));
  L.ml = take(pieces * 2 * 4);
  L.o = take(pieces * c.head_dim * 4);
  L.lse = take(io.mass ? (size_t)L.rows * io.heads * 4 : 0);
  L.scores = take(io.mass ? (size_t)L.rows * io.heads * io.mass_len * 4 : 0);
  L.bytes = at;
  return L;
}

int attend_check(const er_kv_cache* c, const er_kv_attend_io* io) {
  if (int rc = kv_check("er_kv_attend", c)) return rc;
  if (!io) return fail(ER_EINVAL, "er_kv_attend: null io");
  if (io->rows < 0 || io->heads <= 0 || io->heads % c->kv_heads)
    return fail(ER_EINVAL, "er_kv_attend: rows %d, heads %d / %d", io->rows, io->heads, c->kv_heads);
  if (io->q_dtype != ER_DTYPE_F32 && io->q_dtype != ER_DTYPE_BF16)
    return fail(ER_EINVAL, "er_kv_attend: q dtype %d", io->q_dtype);
  if (io->q_stride < (long long)io->heads * c->head_dim)
    return fail(ER_EINVAL, "er_kv_attend: row stride %lld shorter than the queries", io->q_stride);
  if (io->pages && (io->max_pages <= 0 || !io->counts))
    return fail(ER_EINVAL, "er_kv_attend: page lists of %d without counts or room", io->max_pages);
  if (io->pages && io->mass) return fail(ER_EINVAL, "er_kv_attend: mass is not accumulated over page lists");
  if (io->mass && io->mass_len < 0) return fail(ER_EINVAL, "er_kv_attend: mass_len %d", io->mass_len);
  if (!io->seqs && io->rows > c->seqs)
    return fail(ER_EINVAL, "er_kv_attend: %d rows, %d sequences", io->rows, c->seqs);
  if (io->pages && c->kv_heads > kMaxEntries) return fail(ER_EINVAL, "er_kv_attend: %d key heads", c->kv_heads);
  return ER_OK;
}

}  // namespace
}  // namespace er

using namespace er;

extern "C" size_t er_kv_attend_workspace_bytes(const er_kv_cache* cache, const er_kv_attend_io* io) {
  int sms = 0;
  if (attend_check(cache, io) || io->rows == 0 || device_sms(&sms)) return 0;
  return attend_layout(*cache, *io, sms).bytes;
}

extern "C" int er_kv_attend(const er_kv_cache* cache, const er_kv_attend_io* io, void* workspace,
                            size_t workspace_bytes, void* stream) {
  if (int rc = attend_check(cache, io)) return rc;
  if (io->rows == 0) return ER_OK;
  if (!io->q || !io->out || !io->lens) return fail(ER_EINVAL, "er_kv_attend: null pointer");
  int sms = 0;
  if (int rc = device_sms(&sms)) return rc;
  const Layout L = attend_layout(*cache, *io, sms);
  if (L.bytes && (!workspace || workspace_bytes < L.bytes))
    return fail(ER_ENOSPACE, "er_kv_attend: workspace %zu bytes, need %zu", workspace_bytes, L.bytes);
  if ((uintptr_t)workspace & 255) return fail(ER_EINVAL, "er_kv_attend: workspace must be 256-byte aligned");
  cudaStream_t st = (cudaStream_t)stream;
  char* ws = (char*)workspace;
  const size_t qs = io->q_dtype == ER_DTYPE_BF16 ? 2 : 4;
  for (int r0 = 0; r0 < io->rows; r0 += L.rows) {
    AttendArgs a = {};
    a.kv = kv_view(*cache);
    a.rows = io->rows - r0 < L.rows ? io->rows - r0 : L.rows;
    if (!io->seqs) {  // the launch's rows are sequences r0 ..
      a.kv.table += r0 * a.kv.table_stride;
      a.kv.seqs -= r0;
    }
    a.q = (const char*)io->q + (size_t)r0 * io->q_stride * qs;
    a.q_stride = io->q_stride;
    a.out = (char*)io->out + (size_t)r0 * io->heads * cache->head_dim * qs;
    a.heads = io->heads;
    a.group = io->heads / cache->kv_heads;
    a.blocks = L.blocks;
    a.seqs = io->seqs ? io->seqs + r0 : nullptr;
    a.lens = io->lens + r0;
    a.scale = io->scale * 1.4426950408889634f;
    a.max_pages = io->max_pages;
    if (io->pages) {
      a.pages = io->pages + (size_t)r0 * cache->kv_heads * io->max_pages;
      a.counts = io->counts + (size_t)r0 * cache->kv_heads;
    }
    a.tile = L.shape.warps * kKvChunk;
    a.min_share = 2;
    a.status = io->status;
    a.entries = io->pages ? a.rows * cache->kv_heads : a.rows;
    a.units = io->pages ? L.blocks : cache->kv_heads * L.blocks;
    a.cut = (CutUnit*)(ws + L.cut);
    a.part_ml = (float*)(ws + L.ml);
    a.part_o = (float*)(ws + L.o);
    a.grid = L.grid;
    a.cluster = L.cluster;
    if (io->mass) {
      a.lse = (float*)(ws + L.lse);
      a.scores = (float*)(ws + L.scores);
      a.mass = io->mass + r0 * io->mass_row_stride;
      a.mass_row_stride = io->mass_row_stride;
      a.mass_head_stride = io->mass_head_stride;
      a.mass_len = io->mass_len;
    }
    int rc;
    using bf = __nv_bfloat16;
    const bool cb = cache->dtype == ER_DTYPE_BF16, qb = io->q_dtype == ER_DTYPE_BF16;
    if (cb)
      rc = attend_mma(a, io->q_dtype, st);
    else
      rc = qb ? attend_simt<bf>(a, L.shape, st) : attend_simt<float>(a, L.shape, st);
    if (rc) return rc;
    const int gb = L.shape.heads;
    const dim3 grid(L.grid, gb < a.group ? gb : a.group);
    const size_t smem = (size_t)(L.grid + 3) / 4 * 16 + kJoinThreads * 16;
    if (!L.cluster)
    rc = qb ? launch_chained(kv_join_kernel<bf>, grid, dim3(kJoinThreads), smem, st, "kv_join_kernel", a, gb)
            : launch_chained(kv_join_kernel<float>, grid, dim3(kJoinThreads), smem, st, "kv_join_kernel", a, gb);
    if (rc) return rc;
    if (io->mass && io->mass_len > 0) {
      const int pairs = a.rows * cache->kv_heads;
      for (int p0 = 0; p0 < pairs; p0 += 65535 / cache->kv_heads * cache->kv_heads) {
        AttendArgs b = a;  // whole rows at a time: the grid's y extent is 16 bits
        const int r = p0 / cache->kv_heads, n = pairs - p0 < 65535 / cache->kv_heads * cache->kv_heads
                                                    ? pairs - p0
                                                    : 65535 / cache->kv_heads * cache->kv_heads;
        b.lens += r;
        if (b.seqs) {
          b.seqs += r;
        } else {
          b.kv.table += r * b.kv.table_stride;
          b.kv.seqs -= r;
        }
        b.mass += r * b.mass_row_stride;
        b.scores += (size_t)p0 * b.mass_len * b.group;
        b.lse += (size_t)r * b.heads;
        const int most = (io->mass_len + 255) / 256, want = sms * 8 / n + 1;
        rc = launch_chained(kv_mass_kernel, dim3(most < want ? most : want, n), dim3(256), 0, st, "kv_mass_kernel", b);
        if (rc) return rc;
      }
    }
  }
  return ER_OK;
}
