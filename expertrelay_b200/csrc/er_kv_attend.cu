// er_kv_attend.cu -- attention of rows of queries over the paged key-value
// cache: the join of split rows, the accumulated attention weight, and the
// entry point.
#include "er_kv_attend.cuh"

namespace er {

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
    constexpr int N = 12;  // pieces a thread has under way
#pragma unroll 1
    for (int k0 = grp; k0 < n; k0 += groups * N) {
      float4 x[N];
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (k0 + j * groups < n) x[j] = *reinterpret_cast<const float4*>(a.part_o + piece(k0 + j * groups) * d + col * 4);
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (k0 + j * groups < n) fma4(acc, x[j], wt[k0 + j * groups]);
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

// mass[row, h, j] += sum_g 2^(s_gj - lse_g), a thread per position. The scores
// have just been written and lie in L2; what bounds it is latency (7 us beside
// the 62 of the rest at 8 rows of up to 16000 positions, 8 key heads of 4
// queries; four positions of a thread under way at once, or more CTAs, changed
// nothing). A score a load cost 12 us more with 16 queries (54 rows of up to
// 6689 positions, 2 key heads: 90 us, 78).
__global__ void __launch_bounds__(256) kv_mass_kernel(const __grid_constant__ AttendArgs a) {
  kv_enter();
  const int unit = blockIdx.y, row = unit / a.kv.kv_heads, h = unit % a.kv.kv_heads;
  const Entry e = kv_entry(a, row);
  float* to = a.mass + row * a.mass_row_stride + h * a.mass_head_stride;
  if (e.bad) {  // which positions it meant is not known: all are spoilt
    for (long long j = blockIdx.x * 256 + threadIdx.x; j < a.mass_len; j += gridDim.x * 256) to[j] = __int_as_float(0x7fc00000);
    return;
  }
  const float* s = a.scores + (long long)unit * a.mass_len * a.group;
  const float* lse = a.lse + (long long)row * a.heads + h * a.group;
  for (long long j = blockIdx.x * 256 + threadIdx.x; j < e.n; j += gridDim.x * 256) {  // a step may pass 2^31
    float sum = 0.f;
    if (a.group % 4 == 0) {
#pragma unroll 4
      for (int g = 0; g < a.group; g += 4) {
        const float4 x = *reinterpret_cast<const float4*>(s + j * a.group + g);
        sum += exp2f(x.x - lse[g]) + exp2f(x.y - lse[g + 1]) + exp2f(x.z - lse[g + 2]) + exp2f(x.w - lse[g + 3]);
      }
    } else {
#pragma unroll 4
      for (int g = 0; g < a.group; ++g) sum += exp2f(s[j * a.group + g] - lse[g]);
    }
    to[j] += sum;
  }
}

namespace {

// scan entries a launch takes (at least four rows: key heads are 1024 at the most); more rows go in several launches
constexpr int kMaxEntries = 4096;

struct Layout {
  KernelShape shape;
  int blocks, grid, rows;  // rows: of one launch
  bool cluster;
  size_t cut, ml, o, lse, scores, bytes;
};

Layout attend_layout(const er_kv_cache& c, const er_kv_attend_io& io, int sms) {
  Layout L;
  const int group = io.heads / c.kv_heads;
  L.shape = c.dtype == ER_DTYPE_BF16 ? attend_shape_bf16(c.head_dim, group, io.q_dtype)
                                     : attend_shape_f32(c.head_dim, group, io.q_dtype);
  L.blocks = (group + L.shape.heads - 1) / L.shape.heads;
  L.grid = sms * L.shape.per_sm;
  if (L.grid > kJoinThreads * kJoinPieces) L.grid = kJoinThreads * kJoinPieces;
  L.rows = io.pages ? kMaxEntries / c.kv_heads : kMaxEntries;
  if (L.rows > io.rows) L.rows = io.rows;
  if (io.mass) {  // the scores of a launch stay within 256 MB, or one row's
    const long long most = (256ll << 20) / (4ll * io.heads * (io.mass_len > 0 ? io.mass_len : 1));
    if (L.rows > most) L.rows = most < 1 ? 1 : (int)most;
  }
  // A cluster per unit or equal shares of all tiles. The clusters save the
  // division of the line and the join, 4 to 5 us, but a unit has 8 CTAs at most:
  // taken while its longest row gives each of those at most 120 KB of keys and
  // values more than a share would be (they take in 25 GB/s each), and all
  // clusters run at once. (One row of 2000 positions, by clusters and by shares:
  // 8 key heads of 64, bf16 8.8 and 11.7 us; of 128 10.5 and 11.5; 16 of 128, fp32
  // 18.5 and 16.3. Of 5000, before bf16 results had weights of three parts: 11.9
  // and 12.6; 18.1 and 13.3; 35.9 and 28.1.) It takes two CTAs an SM: with one,
  // 16 clusters of 8 did not all find room in the processor clusters of 148 SMs,
  // and went in two waves.
  const long long units = (long long)L.rows * c.kv_heads * L.blocks, ctas = L.grid, most = kKvMaxLen;
  const long long room = (io.pages ? (long long)io.max_pages : (long long)c.table_width) * c.page_size;
  const long long bytes = (room < most ? room : most) * 2 * c.head_dim * (c.dtype == ER_DTYPE_BF16 ? 2 : 4);
  L.cluster = L.rows == io.rows && L.shape.per_sm >= 2 && units * kClusterCtas <= ctas &&
              bytes / kClusterCtas * (ctas - units * kClusterCtas) <= (120ll << 10) * ctas;
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
  if (io->rows < 0 || io->heads <= 0 || io->heads > kMaxHeads || io->heads % c->kv_heads)
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
  if ((uintptr_t)io->out & 15) return fail(ER_EINVAL, "er_kv_attend: out must be 16-byte aligned");
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
    a.tile = L.shape.tile;
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
    const bool qb = io->q_dtype == ER_DTYPE_BF16;
    rc = cache->dtype == ER_DTYPE_BF16 ? attend_bf16(a, io->q_dtype, st) : attend_f32(a, io->q_dtype, st);
    if (rc) return rc;
    const int gb = L.shape.heads;
    const dim3 grid(L.grid, gb < a.group ? gb : a.group);
    const size_t smem = (size_t)(L.grid + 3) / 4 * 16 + kJoinThreads * 16;
    if (!L.cluster) {
      rc = qb ? launch_chained(kv_join_kernel<bf>, grid, dim3(kJoinThreads), smem, st, "kv_join_kernel", a, gb)
              : launch_chained(kv_join_kernel<float>, grid, dim3(kJoinThreads), smem, st, "kv_join_kernel", a, gb);
      if (rc) return rc;
    }
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
