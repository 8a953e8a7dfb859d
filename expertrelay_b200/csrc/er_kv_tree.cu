// er_kv_tree.cu -- attention of a tree of drafted tokens over a paged cache.
#include "er_kv_tree.cuh"
#include "er_ptx.cuh"

namespace er {

namespace {

// Joins the units that several CTAs share: CTA (x, y) takes every gridDim.x-th
// of them from x on, of its rows every gridDim.y-th. Of many pieces the warps
// share a row's, of few each takes rows of its own. Also writes the rows of
// trees that something is wrong with, which no attention CTA meets, and of all
// trees where an attention CTA gave up.
constexpr int kJoinWarps = 8, kJoinMost = 1024;  // CTAs that may share a line at most

template <typename TQ>
__global__ void __launch_bounds__(kJoinWarps * 32, 3) kv_tree_join_kernel(const __grid_constant__ TreeArgs a) {
  __shared__ int cuts[kJoinMost], found;
  __shared__ float4 sums[kJoinWarps][32];
  __shared__ float2 tops[kJoinWarps];
  kv_enter();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, d = a.kv.d;
  auto spoil = [&](bool all) {
    for (int t = blockIdx.y * gridDim.x + blockIdx.x; t < a.trees; t += gridDim.x * gridDim.y) {
      const Tree e = kv_tree(a, t);
      if (!e.bad && !all) continue;
      TQ* out = (TQ*)a.out + (long long)e.first * a.heads * d;
      for (long long i = threadIdx.x; i < (long long)e.nodes * a.heads * d; i += kJoinWarps * 32)
        out[i] = kv_round<TQ>(__int_as_float(0x7fc00000));
    }
  };
  spoil(false);  // beside the other warps' look at the cuts
  if (warp == 0) {  // the CTAs in whose runs such a unit begins
    int n = 0;
    bool gave_up = false;
    for (int c0 = 0; c0 < a.grid; c0 += 32) {
      const int live = c0 + lane < a.grid ? a.cut[c0 + lane].live : 0;
      const uint32_t all = __ballot_sync(0xffffffffu, live > 0);
      if (live > 0) cuts[n + __popc(all & ((1u << lane) - 1))] = c0 + lane;
      n += __popc(all);
      gave_up |= live < 0;
    }
    gave_up = __any_sync(0xffffffffu, gave_up);
    if (lane == 0) found = gave_up ? -1 : n;
  }
  __syncthreads();
  if (found < 0) spoil(true);
  constexpr int N = 8;  // pieces under way
#pragma unroll 1
  for (int f = blockIdx.x; f < found; f += gridDim.x) {
    const int i0 = cuts[f];
    const TreeCut c = a.cut[i0];
    const int n = kv_share_of(c.total, tree_shares(a, c.total), c.begin + a.unit_cost + c.tiles - 1) - i0 + 1;  // pieces
    const bool together = n > 2 * N;
    const int step = together ? gridDim.y : gridDim.y * kJoinWarps, k1 = together ? warp : 0, by = together ? kJoinWarps : 1;
    const int width = min(a.channels, d - c.ch0);
    const bool mine = lane * 4 < width;
#pragma unroll 1
    for (int r = together ? blockIdx.y : blockIdx.y * kJoinWarps + warp; r < c.live; r += step) {
      auto at = [&](int k) { return ((long long)(i0 + k) * 2 + (k == 0 ? 1 : 0)) * a.piece_rows + r; };
      float top = -INFINITY;
      for (int k = k1 + lane * by; k < n; k += 32 * by) top = fmaxf(top, a.part_ml[at(k) * 2]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      float sum = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
      for (int k0 = k1; k0 < n; k0 += N * by) {
        float2 ml[N];
        float4 x[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
          if (k0 + j * by >= n) continue;
          ml[j] = *reinterpret_cast<const float2*>(a.part_ml + at(k0 + j * by) * 2);
          if (mine) x[j] = *reinterpret_cast<const float4*>(a.part_o + at(k0 + j * by) * a.channels + lane * 4);
        }
#pragma unroll
        for (int j = 0; j < N; ++j) {
          if (k0 + j * by >= n) continue;
          const float weight = piece_weight(ml[j].x, top);
          sum = fmaf(ml[j].y, weight, sum);  // a spoilt piece's sum is NaN
          if (mine) fma4(acc, x[j], weight);
        }
      }
      if (together) {
        __syncthreads();
        sums[warp][lane] = acc;
        if (lane == 0) tops[warp] = make_float2(top, sum);
        __syncthreads();
        if (warp > 0) continue;
        for (int i = 1; i < kJoinWarps; ++i) top = fmaxf(top, tops[i].x);
        acc = make_float4(0.f, 0.f, 0.f, 0.f);
        sum = 0.f;
        for (int i = 0; i < kJoinWarps; ++i) {
          const float weight = piece_weight(tops[i].x, top);
          sum = fmaf(tops[i].y, weight, sum);
          fma4(acc, sums[i][lane], weight);
        }
      }
      const int q = c.q0 + r, node = tree_node(a, q), g = q - node * a.group;
      if (mine)
        kv_store4((TQ*)a.out + ((long long)(c.first + node) * a.heads + c.head * a.group + g) * d + c.ch0 + lane * 4, acc, sum);
    }
  }
}

int tree_check(const er_kv_cache* c, const er_kv_tree_io* io) {
  if (int rc = kv_check("er_kv_tree", c)) return rc;
  if (!io) return fail(ER_EINVAL, "er_kv_tree: null io");
  if (io->rows < 0 || io->trees < 0 || io->heads <= 0 || io->heads > kMaxHeads || io->heads % c->kv_heads)
    return fail(ER_EINVAL, "er_kv_tree: %d rows of %d trees, heads %d / %d", io->rows, io->trees, io->heads, c->kv_heads);
  if (io->trees > kMaxTrees) return fail(ER_EINVAL, "er_kv_tree: %d trees (at most %d)", io->trees, kMaxTrees);
  if (io->q_dtype != ER_DTYPE_F32 && io->q_dtype != ER_DTYPE_BF16)
    return fail(ER_EINVAL, "er_kv_tree: q dtype %d", io->q_dtype);
  if (io->q_stride < (long long)io->heads * c->head_dim)
    return fail(ER_EINVAL, "er_kv_tree: row stride %lld shorter than the queries", io->q_stride);
  if (!io->seqs && io->trees > c->seqs)
    return fail(ER_EINVAL, "er_kv_tree: %d trees, %d sequences", io->trees, c->seqs);
  return ER_OK;
}

}  // namespace
}  // namespace er

using namespace er;

namespace {

// er_kv_tree_test_stall: the limit of a wait, and whether the attention kernel's CTAs end with one that runs out
unsigned long long tree_wait_ns = kDefaultWaitNs;
int tree_stall = 0;

struct TreeLayout {
  TreeLaunch shape;
  int piece_rows;
  size_t cut, ml, o, bytes;
};

TreeLayout tree_layout(const er_kv_cache& c, const er_kv_tree_io& io, int sms) {
  TreeLayout L;
  const int group = io.heads / c.kv_heads;
  L.shape = c.dtype == ER_DTYPE_BF16 ? tree_shape_bf16(c.head_dim, io.q_dtype) : tree_shape_f32(c.head_dim);
  const long long rows = (long long)(io.rows < kMaxNodes ? io.rows : kMaxNodes) * group;
  L.piece_rows = rows < L.shape.rows ? (int)rows : L.shape.rows;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += align_up(bytes, 256);
    return here;
  };
  const size_t n = (size_t)sms * 2 * L.piece_rows;
  L.cut = take(sms * sizeof(TreeCut));
  L.ml = take(n * 8);
  L.o = take(n * L.shape.channels * 4);
  L.bytes = at;
  return L;
}

// Pages of a pool as copies see them: channels, positions, key heads, pages. bf16: boxes of 64 channels, as the
// products want them (128-byte swizzle), fp32: rows as they are.
int tree_map(CUtensorMap* m, const er_kv_cache& c, void* pool, int box_rows, int box_channels) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(ER_ECUDA, "cuTensorMapEncodeTiled is not available from the driver");
  const bool half = c.dtype == ER_DTYPE_BF16;
  const cuuint64_t es = half ? 2 : 4;
  const cuuint64_t dims[4] = {(cuuint64_t)c.head_dim, (cuuint64_t)c.page_size, (cuuint64_t)c.kv_heads, (cuuint64_t)c.num_pages};
  cuuint64_t strides[3] = {(cuuint64_t)c.slot_stride * es, (cuuint64_t)c.head_stride * es, (cuuint64_t)c.page_stride * es};
  for (int i = 0; i < 3; ++i)
    if (dims[i + 1] == 1) strides[i] = (cuuint64_t)c.head_dim * es;  // never used
  const cuuint32_t box[4] = {(cuuint32_t)box_channels, (cuuint32_t)box_rows, 1, 1}, each[4] = {1, 1, 1, 1};
  const CUresult r = fn(m, half ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, pool, dims, strides,
                        box, each, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        half ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(ER_EINVAL, "er_kv_tree: pools of strides %lld, %lld, %lld cannot be copied by tiles (%d)", c.page_stride,
                c.head_stride, c.slot_stride, (int)r);
  return ER_OK;
}

}  // namespace

extern "C" size_t er_kv_tree_workspace_bytes(const er_kv_cache* cache, const er_kv_tree_io* io) {
  int sms = 0;
  if (tree_check(cache, io) || io->rows == 0 || io->trees == 0 || device_sms(&sms)) return 0;
  return tree_layout(*cache, *io, sms).bytes;
}

extern "C" int er_kv_tree(const er_kv_cache* cache, const er_kv_tree_io* io, void* workspace, size_t workspace_bytes,
                          void* stream) {
  if (int rc = tree_check(cache, io)) return rc;
  if (io->rows == 0 || io->trees == 0) return ER_OK;
  if (!io->q || !io->out || !io->lens || !io->starts || !io->parents)
    return fail(ER_EINVAL, "er_kv_tree: null pointer");
  if ((uintptr_t)io->out & 15) return fail(ER_EINVAL, "er_kv_tree: out must be 16-byte aligned");
  // A unit's queries are read by its own CTAs alone, and before its rows are written: results may take the place of
  // their own queries, but for heads that two units share.
  const long long each = (long long)io->heads * cache->head_dim, es = io->q_dtype == ER_DTYPE_BF16 ? 2 : 4;
  const uintptr_t q = (uintptr_t)io->q, out = (uintptr_t)io->out;
  if (q < out + io->rows * each * es && out < q + ((io->rows - 1) * io->q_stride + each) * es &&
      (q != out || (io->rows > 1 && io->q_stride != each) || cache->head_dim > kTreeChannels))
    return fail(ER_EINVAL, "er_kv_tree: q and out share memory (only the same rows may, of at most %d channels a head)",
                kTreeChannels);
  int sms = 0;
  if (int rc = device_sms(&sms)) return rc;
  if (sms > kJoinMost) sms = kJoinMost;
  const TreeLayout L = tree_layout(*cache, *io, sms);
  if (!workspace || workspace_bytes < L.bytes)
    return fail(ER_ENOSPACE, "er_kv_tree: workspace %zu bytes, need %zu", workspace_bytes, L.bytes);
  if ((uintptr_t)workspace & 255) return fail(ER_EINVAL, "er_kv_tree: workspace must be 256-byte aligned");
  cudaStream_t st = (cudaStream_t)stream;
  char* ws = (char*)workspace;
  TreeArgs a = {};
  a.kv = kv_view(*cache);
  a.q = io->q, a.q_stride = io->q_stride, a.out = io->out;
  a.rows = io->rows, a.heads = io->heads, a.group = io->heads / cache->kv_heads, a.trees = io->trees;
  a.starts = io->starts, a.parents = io->parents, a.seqs = io->seqs, a.lens = io->lens;
  // positive in the kernel, so that the greatest product has the greatest score
  a.q_flip = io->scale < 0.f, a.q_zero = io->scale == 0.f;
  a.scale = (a.q_zero ? 1.f : a.q_flip ? -io->scale : io->scale) * 1.4426950408889634f;
  a.status = io->status;
  using bf = __nv_bfloat16;
  const bool qb = io->q_dtype == ER_DTYPE_BF16, cb = cache->dtype == ER_DTYPE_BF16;
  const long long qs = qb ? 2 : 4;
  a.q_wide = (((uintptr_t)io->q | (uintptr_t)(io->q_stride * qs)) & 15) == 0;
  a.grid = sms;
  a.piece_rows = L.piece_rows;
  a.cut = (TreeCut*)(ws + L.cut);
  a.part_ml = (float*)(ws + L.ml);
  a.part_o = (float*)(ws + L.o);
  while (1 << a.tile_shift < L.shape.tile) ++a.tile_shift;
  while (1 << a.block_shift < L.shape.rows) ++a.block_shift;
  // 24 trees of up to 4097 positions, 16 heads, bf16: 4 tiles 147 us, 8 141, 14 139, 24 140; 6 of up to 2500, fp32,
  // whose tiles take four times as long: 150, 151, 157 and 169
  a.unit_cost = cb ? 12 : 4;
  a.wait_ns = tree_wait_ns, a.stall = tree_stall;
  a.block_rows = L.shape.rows, a.channels = L.shape.channels, a.halves = L.shape.halves;
  CUtensorMap maps[2] = {};
  if (L.shape.box_rows) {
    a.box_rows = L.shape.box_rows;
    while (cache->page_size % a.box_rows) a.box_rows >>= 1;
    if (int rc = tree_map(&maps[0], *cache, cache->k, a.box_rows, L.shape.box_channels)) return rc;
    if (int rc = tree_map(&maps[1], *cache, cache->v, a.box_rows, L.shape.box_channels)) return rc;
  }
  if (int rc = cb ? tree_bf16(a, io->q_dtype, maps, st) : tree_f32(a, io->q_dtype, maps, st)) return rc;
  // few units: many pieces each, and a CTA a row for them
  const long long blocks = ((long long)(io->rows < kMaxNodes ? io->rows : kMaxNodes) * a.group + a.block_rows - 1) / a.block_rows;
  const long long units = (long long)io->trees * cache->kv_heads * blocks * a.halves;
  const int across = units < sms ? (int)units : sms;
  int parts = 4 * sms / across;
  if (parts > L.piece_rows) parts = L.piece_rows;
  const dim3 grid(across, parts);
  return qb ? kv_launch(kv_tree_join_kernel<bf>, grid, kJoinWarps * 32, 0, false, st, "kv_tree_join_kernel", a)
            : kv_launch(kv_tree_join_kernel<float>, grid, kJoinWarps * 32, 0, false, st, "kv_tree_join_kernel", a);
}

extern "C" int er_kv_tree_test_stall(unsigned long long wait_ns, int stall) {
  if (stall < 0 || stall > 1) return fail(ER_EINVAL, "er_kv_tree_test_stall: stall %d (0 or 1)", stall);
  tree_wait_ns = wait_ns ? wait_ns : kDefaultWaitNs;
  tree_stall = stall;
  return ER_OK;
}
