// er_kv_pages.cu -- pages and places of a paged cache moved about, all layers
// in one launch: copies of pages (forks of sequences, a pool's pages moved
// together) and the compaction of a sequence's places (an accepted path of a
// draft, a text that lost a part).
#include "er_kv.cuh"

namespace er {

namespace {

// Both pools of every layer: layer l's page p begins at l * layer_stride + p * page_stride (bytes).
struct Layers {
  KvView kv;
  long long layer_stride;
  int layers, row16;  // 16-byte vectors of a slot's head_dim values
};

__device__ __forceinline__ uint4 load16(const char* p) { return *reinterpret_cast<const uint4*>(p); }
__device__ __forceinline__ void store16(char* p, uint4 v) { *reinterpret_cast<uint4*>(p) = v; }

constexpr int kThreads = 256, kMany = 8;  // vectors a thread has under way

struct CopyArgs {
  Layers l;
  const int32_t *src, *dst, *used;
  int n;
  int* status;
};

// out page = in page, the used slots of it: twice their bytes, which bounds it
// (500 pages of 128 KB of keys and as many of values in 8 layers: 320 us, 6.55 TB/s;
// 4 partly filled pages in 24 layers, 142 MB in all: 25 us, 0.87 of that).
// Grid (parts of a page, 2 layers, pairs). A page's used slots are rows of
// runs: whole pages that are contiguous are one run, pages of contiguous heads
// a run a head, other layouts a run a slot of one head.
__global__ void __launch_bounds__(kThreads) kv_copy_pages_kernel(const __grid_constant__ CopyArgs a) {
  kv_enter();
  const KvView& kv = a.l.kv;
#pragma unroll 1
  for (int pair = blockIdx.z; pair < a.n; pair += gridDim.z) {
    const int from = a.src[pair], to = a.dst[pair], used = a.used ? a.used[pair] : kv.page_size;
    if (from < 0) continue;
    const int bad = from >= kv.num_pages || to < 0 || to >= kv.num_pages ? ER_KV_BAD_PAGE
                    : used < 0 || used > kv.page_size                     ? ER_KV_BAD_LENGTH
                                                                          : 0;
    if (bad) {
      if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) kv_report(a.status, bad);
      continue;
    }
    const int row16 = a.l.row16, layer = blockIdx.y >> 1;
    char* pool = (blockIdx.y & 1 ? kv.v : kv.k) + layer * a.l.layer_stride;
    const char* s = pool + from * kv.page_stride;
    char* d = pool + to * kv.page_stride;
    // vectors of a run, and runs: `runs1` of them stride1 apart, over and over stride2 apart
    const bool slots = kv.slot_stride == row16 * 16ll, heads = kv.head_stride == row16 * 16ll;
    int run = row16, runs1, runs2;
    long long stride1, stride2;
    if (slots) {
      run *= used, runs1 = kv.kv_heads, runs2 = 1, stride1 = kv.head_stride, stride2 = 0;
      if (stride1 == run * 16ll) run *= runs1, runs1 = 1;
    } else if (heads) {
      run *= kv.kv_heads, runs1 = used, runs2 = 1, stride1 = kv.slot_stride, stride2 = 0;
      if (stride1 == run * 16ll) run *= runs1, runs1 = 1;
    } else {
      runs1 = used, runs2 = kv.kv_heads, stride1 = kv.slot_stride, stride2 = kv.head_stride;
    }
    const int total = run * runs1 * runs2;
    const int step = gridDim.x * kThreads * kMany;
#pragma unroll 1
    for (int i0 = blockIdx.x * kThreads * kMany + threadIdx.x; i0 < total; i0 += step) {
      uint4 v[kMany];
      long long at[kMany];
#pragma unroll
      for (int j = 0; j < kMany; ++j) {
        const int i = i0 + j * kThreads;
        if (i >= total) continue;
        const int r = run == total ? 0 : i / run, in = i - r * run;
        const int r2 = runs2 == 1 ? 0 : r / runs1, r1 = r - r2 * runs1;
        at[j] = r2 * stride2 + r1 * stride1 + in * 16ll;
        v[j] = load16(s + at[j]);
      }
#pragma unroll
      for (int j = 0; j < kMany; ++j)
        if (i0 + j * kThreads < total) store16(d + at[j], v[j]);
    }
  }
}

struct CompactArgs {
  Layers l;
  const int32_t *seqs, *start, *keep, *counts;
  int rows, most;    // most: entries of a row's list
  long long keep_stride;
  int heads, cuts;   // of one CTA: key heads, or one of so many parts of a head's channels
  int32_t* lens_out;
  int* status;
};

// Grid (columns, 2 layers, rows). Place start + keep[j] goes to start + j. keep
// ascends, so keep[j] >= j: what is written at j is read only for entries up to
// j, and a CTA that takes the list in order, loading a batch before it stores
// it, needs no second copy. Batches cannot be shared between CTAs that way, so
// a CTA takes as few columns as keep its threads busy: several key heads of a
// short list, 128 bytes of one head of a long one (twelve lists of up to 1501
// places, 490 MB in all: 114 us, with whole heads 125, with 64 bytes 118). DRAM
// bounds it; the last CTAs are those of the shortest lists (104 us, 4.7 TB/s:
// before and behind a batch's barrier only loads or only stores are under way).
// An accepted draft's 5 places in 24 layers: 5.5 us, latency.
constexpr int kBatchRows = 512, kCut = 8;  // kCut: vectors of a place a CTA has at least

__global__ void __launch_bounds__(kThreads) kv_compact_kernel(const __grid_constant__ CompactArgs a) {
  kv_enter();
  __shared__ long long from[3][kBatchRows], to[3][kBatchRows];
  const KvView& kv = a.l.kv;
  const int layer = blockIdx.y >> 1, column = blockIdx.x / a.cuts, row16 = a.l.row16 / a.cuts;
  const int h0 = column * a.heads, heads = min(a.heads, kv.kv_heads - h0);
  char* pool = (blockIdx.y & 1 ? kv.v : kv.k) + layer * a.l.layer_stride + h0 * kv.head_stride +
               (blockIdx.x - column * a.cuts) * row16 * 16;
  const int width = heads * row16;  // vectors of a place
  const int batch = min(kBatchRows, kThreads * kMany / width);
  int z = blockIdx.z;
  if (a.rows > 1 && a.rows <= kThreads) {  // the longest lists first
    __shared__ int all[kThreads], which;
    const int mine = (int)threadIdx.x < a.rows ? a.counts[threadIdx.x] : 0;
    all[threadIdx.x] = mine;
    __syncthreads();
    if ((int)threadIdx.x < a.rows) {
      int rank = 0;
      for (int i = 0; i < a.rows; ++i) rank += all[i] > mine || (all[i] == mine && i < (int)threadIdx.x);
      if (rank == z) which = threadIdx.x;
    }
    __syncthreads();
    z = which;
  }
#pragma unroll 1
  for (int row = z; row < a.rows; row += gridDim.z) {
    const int seq = a.seqs ? a.seqs[row] : row, start = a.start[row], n = a.counts[row];
    const int32_t* keep = a.keep + row * a.keep_stride;
    int bad = 0;
    if (seq < 0 || seq >= kv.seqs)
      bad = ER_KV_BAD_SEQ;
    else if (n < 0 || n > a.most || start < 0 || start > kv.capacity())
      bad = ER_KV_BAD_LENGTH;
    const int32_t* pages = bad ? nullptr : kv.pages_of(seq);
    // the whole list before anything is written: every CTA of the row finds the same
    for (int j = threadIdx.x; !bad && j < n; j += kThreads) {
      const int k = keep[j], before = j ? keep[j - 1] : -1;
      if (k <= before || (long long)start + k >= min(kv.capacity(), 0x7fffffffll)) {  // places stay ints
        bad = ER_KV_BAD_LENGTH;
      } else {
        const int p = pages[kv.ordinal(start + k)], q = pages[kv.ordinal(start + j)];
        if (p < 0 || p >= kv.num_pages || q < 0 || q >= kv.num_pages) bad = ER_KV_BAD_PAGE;
      }
    }
    const bool first = blockIdx.x == 0 && blockIdx.y == 0, spoilt = __syncthreads_or(bad);
    if (first && bad) kv_report(a.status, bad);
    if (first && threadIdx.x == 0 && a.lens_out) a.lens_out[row] = spoilt ? -1 : start + n;
    if (spoilt || n == 0) continue;
    auto look = [&](int j0, int b) {
      for (int r = threadIdx.x; r < batch && j0 + r < n; r += kThreads) {
        const int p = start + keep[j0 + r], q = start + j0 + r;
        from[b][r] = pages[kv.ordinal(p)] * kv.page_stride + kv.slot(p) * kv.slot_stride;
        to[b][r] = pages[kv.ordinal(q)] * kv.page_stride + kv.slot(q) * kv.slot_stride;
      }
    };
    look(0, 0);
    __syncthreads();
    // Places in three buffers, for one barrier a batch: the places that batch i + 1 gets were batch i - 2's. Those were
    // read last by i - 2's stores, before a thread's barrier of batch i - 1, and are written behind that barrier. In two
    // they would be batch i - 1's, which a warp behind the others may still have to read for its stores.
    int b = 0;
#pragma unroll 1
    for (int j0 = 0; j0 < n; j0 += batch) {
      const int following = b == 2 ? 0 : b + 1;
      const int total = min(batch, n - j0) * width;
      uint4 v[kMany];
#pragma unroll
      for (int u = 0; u < kMany; ++u) {
        const int i = threadIdx.x + u * kThreads;
        if (i >= total) continue;
        const int r = i / width, c = i - r * width, h = c / row16;
        v[u] = load16(pool + from[b][r] + h * kv.head_stride + (c - h * row16) * 16);
      }
      if (j0 + batch < n) look(j0 + batch, following);
      __syncthreads();  // all of the batch is read, and the next one's places are known
#pragma unroll
      for (int u = 0; u < kMany; ++u) {
        const int i = threadIdx.x + u * kThreads;
        if (i >= total) continue;
        const int r = i / width, c = i - r * width, h = c / row16;
        store16(pool + to[b][r] + h * kv.head_stride + (c - h * row16) * 16, v[u]);
      }
      b = following;
    }
    __syncthreads();  // the places of the last batch are used no more
  }
}

int layers_of(const char* who, const er_kv_cache* c, int layers, long long layer_stride, Layers* out) {
  if (int rc = kv_check(who, c)) return rc;
  const long long es = c->dtype == ER_DTYPE_BF16 ? 2 : 4;
  if (layers <= 0 || layers > 32767) return fail(ER_EINVAL, "%s: %d layers (1 to 32767)", who, layers);
  if ((layer_stride * es) & 15) return fail(ER_EINVAL, "%s: layers must lie on 16-byte boundaries", who);
  out->kv = kv_view(*c);
  out->layer_stride = layer_stride * es;
  out->layers = layers;
  out->row16 = (int)(c->head_dim * es / 16);
  if ((long long)c->kv_heads * c->page_size * out->row16 > 0x40000000ll)
    return fail(ER_EINVAL, "%s: pages of %d positions, %d key heads: above 16 GB", who, c->page_size, c->kv_heads);
  return ER_OK;
}

}  // namespace
}  // namespace er

using namespace er;

extern "C" int er_kv_copy_pages(const er_kv_cache* cache, int layers, long long layer_stride, const int32_t* src,
                                const int32_t* dst, const int32_t* used, int n, int* status, void* stream) {
  CopyArgs a = {};
  if (int rc = layers_of("er_kv_copy_pages", cache, layers, layer_stride, &a.l)) return rc;
  if (n < 0) return fail(ER_EINVAL, "er_kv_copy_pages: n %d", n);
  if (n == 0) return ER_OK;
  if (!src || !dst) return fail(ER_EINVAL, "er_kv_copy_pages: null pointer");
  a.src = src, a.dst = dst, a.used = used, a.n = n, a.status = status;
  const long long vectors = (long long)cache->kv_heads * cache->page_size * a.l.row16;
  const int parts = (int)((vectors + kThreads * kMany - 1) / (kThreads * kMany));
  return kv_launch(kv_copy_pages_kernel, dim3(parts, 2 * layers, n < 65535 ? n : 65535), kThreads, 0, false,
                   (cudaStream_t)stream, "kv_copy_pages_kernel", a);
}

extern "C" int er_kv_compact(const er_kv_cache* cache, int layers, long long layer_stride, const int32_t* seqs,
                             const int32_t* start, const int32_t* keep, long long keep_stride, int most,
                             const int32_t* counts, int rows, int32_t* lens_out, int* status, void* stream) {
  CompactArgs a = {};
  if (int rc = layers_of("er_kv_compact", cache, layers, layer_stride, &a.l)) return rc;
  if (rows < 0 || most < 0 || keep_stride < most)
    return fail(ER_EINVAL, "er_kv_compact: %d rows of %d entries, stride %lld", rows, most, keep_stride);
  if (!seqs && rows > cache->seqs)
    return fail(ER_EINVAL, "er_kv_compact: %d rows, %d sequences", rows, cache->seqs);
  if (rows == 0) return ER_OK;
  if (!start || !counts || (most > 0 && !keep)) return fail(ER_EINVAL, "er_kv_compact: null pointer");
  // one CTA of a row writes its length when others may not have read what the row is to do
  auto meets = [&](const int32_t* p, long long n) { return p && lens_out && p < lens_out + rows && lens_out < p + n; };
  if (meets(start, rows) || meets(counts, rows) || meets(seqs, rows) || meets(keep, (rows - 1) * keep_stride + most))
    return fail(ER_EINVAL, "er_kv_compact: lens_out shares memory with what the call reads");
  a.seqs = seqs, a.start = start, a.keep = keep, a.counts = counts, a.rows = rows, a.most = most;
  a.keep_stride = keep_stride, a.lens_out = lens_out, a.status = status;
  const long long fill = (long long)kThreads * kMany / ((long long)(most ? most : 1) * a.l.row16);
  a.heads = fill < 1 ? 1 : fill > cache->kv_heads ? cache->kv_heads : (int)fill;
  if (a.heads > kThreads * kMany / a.l.row16) a.heads = kThreads * kMany / a.l.row16;
  a.cuts = 1;
  if (fill < 1)
    while (a.l.row16 % (2 * a.cuts) == 0 && a.l.row16 / (2 * a.cuts) >= kCut) a.cuts *= 2;
  const int blocks = (cache->kv_heads + a.heads - 1) / a.heads * a.cuts;
  return kv_launch(kv_compact_kernel, dim3(blocks, 2 * layers, rows < 65535 ? rows : 65535), kThreads, 0, false,
                   (cudaStream_t)stream, "kv_compact_kernel", a);
}
