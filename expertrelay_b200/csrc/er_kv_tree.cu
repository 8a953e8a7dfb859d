// er_kv_tree.cu -- attention of a tree of drafted tokens over a paged cache.
#include "er_kv_attend.cuh"
#include "er_kv_tree.cuh"

namespace er {

namespace {

// A CTA a (node, head): its warps take every fourth key.
template <typename TC, typename TQ>
__global__ void __launch_bounds__(128) kv_tree_simple_kernel(const __grid_constant__ TreeArgs a) {
  kv_enter();
  __shared__ float part[4][2 + 256];
  __shared__ int find[2], bad_page;
  const int row = blockIdx.x, head = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, d = a.kv.d;
  if (threadIdx.x == 0) find[0] = -1, bad_page = 0;
  __syncthreads();
  for (int t = threadIdx.x; t < a.trees; t += 128) {
    const Tree e = kv_tree(a, t);
    if (e.bad && blockIdx.x == 0 && blockIdx.y == 0) kv_report(a.status, e.bad);
    if (row >= e.first && row < e.first + e.nodes) find[0] = t;
  }
  __syncthreads();
  if (find[0] < 0) return;
  const Tree e = kv_tree(a, find[0]);
  int bad = e.bad;
  if (!bad) {
    for (int i = threadIdx.x; i < e.nodes; i += 128) {
      const int p = a.parents[e.first + i];
      if (p < -1 || p >= i) bad = ER_KV_BAD_TREE;
    }
  }
  if (bad) kv_report(a.status, bad);
  bad = __syncthreads_or(bad);
  TQ* out = (TQ*)a.out + ((long long)row * a.heads + head) * d;
  if (bad) {
    for (int c = threadIdx.x; c < d; c += 128) out[c] = kv_round<TQ>(__int_as_float(0x7fc00000));
    return;
  }
  const TQ* q = (const TQ*)a.q + (long long)row * a.q_stride + (long long)head * d;
  const int h = head / a.group, node = row - e.first;
  float x[8], o[8], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    x[j] = lane + 32 * j < d ? to_f32(q[lane + 32 * j]) * a.scale : 0.f;
    o[j] = 0.f;
  }
  const int32_t* pages = a.kv.pages_of(e.seq);
  for (int j = warp; j < e.len + e.nodes; j += 4) {
    const int pg = pages[a.kv.ordinal(j)];
    if (pg < 0 || pg >= a.kv.num_pages) {
      bad_page = 1;
      continue;
    }
    if (j >= e.len) {
      int at = node;
      while (at > j - e.len) at = a.parents[e.first + at];
      if (at != j - e.len) continue;
    }
    const long long off = pg * a.kv.page_stride + h * a.kv.head_stride + a.kv.slot(j) * a.kv.slot_stride;
    const TC *k = (const TC*)(a.kv.k + off), *v = (const TC*)(a.kv.v + off);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < d) s = fmaf(x[i], to_f32(k[lane + 32 * i]), s);
    s = warp_sum(s);
    if (s == -INFINITY) continue;
    const float top = fmaxf(m, s), by = piece_weight(m, top), p = exp2f(s - top);
    m = top;
    l = l * by + p;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < d) o[i] = o[i] * by + p * to_f32(v[lane + 32 * i]);
  }
  if (lane == 0) part[warp][0] = m, part[warp][1] = l;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (lane + 32 * i < d) part[warp][2 + lane + 32 * i] = o[i];
  __syncthreads();
  float top = -INFINITY, sum = 0.f;
  for (int w = 0; w < 4; ++w) top = fmaxf(top, part[w][0]);
  for (int w = 0; w < 4; ++w) sum += part[w][1] * piece_weight(part[w][0], top);
  if (bad_page && threadIdx.x == 0) kv_report(a.status, ER_KV_BAD_PAGE);
  for (int c = threadIdx.x; c < d; c += 128) {
    float v = 0.f;
    for (int w = 0; w < 4; ++w) v += part[w][2 + c] * piece_weight(part[w][0], top);
    v = sum == 0.f ? 0.f : v / sum;
    out[c] = kv_round<TQ>(bad_page ? __int_as_float(0x7fc00000) : v);
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

extern "C" size_t er_kv_tree_workspace_bytes(const er_kv_cache* cache, const er_kv_tree_io* io) {
  if (tree_check(cache, io)) return 0;
  return 0;
}

extern "C" int er_kv_tree(const er_kv_cache* cache, const er_kv_tree_io* io, void* workspace, size_t workspace_bytes,
                          void* stream) {
  (void)workspace, (void)workspace_bytes;
  if (int rc = tree_check(cache, io)) return rc;
  if (io->rows == 0 || io->trees == 0) return ER_OK;
  if (!io->q || !io->out || !io->lens || !io->starts || !io->parents)
    return fail(ER_EINVAL, "er_kv_tree: null pointer");
  if ((uintptr_t)io->out & 15) return fail(ER_EINVAL, "er_kv_tree: out must be 16-byte aligned");
  TreeArgs a = {};
  a.kv = kv_view(*cache);
  a.q = io->q, a.q_stride = io->q_stride, a.out = io->out;
  a.rows = io->rows, a.heads = io->heads, a.group = io->heads / cache->kv_heads, a.trees = io->trees;
  a.starts = io->starts, a.parents = io->parents, a.seqs = io->seqs, a.lens = io->lens;
  a.scale = io->scale * 1.4426950408889634f;
  a.status = io->status;
  using bf = __nv_bfloat16;
  const bool qb = io->q_dtype == ER_DTYPE_BF16, cb = cache->dtype == ER_DTYPE_BF16;
  auto kernel = cb ? (qb ? kv_tree_simple_kernel<bf, bf> : kv_tree_simple_kernel<bf, float>)
                   : (qb ? kv_tree_simple_kernel<float, bf> : kv_tree_simple_kernel<float, float>);
  return kv_launch(kernel, dim3(io->rows, io->heads), 128, 0, false, (cudaStream_t)stream, "kv_tree_kernel", a);
}
