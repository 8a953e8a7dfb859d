// er_kv_tree_mma.cuh -- tree attention on the tensor cores (tcgen05).
//
// out_i = sum_j 2^(s_ij - m_i) v_j / sum_j 2^(s_ij - m_i), s = scale log2(e) q k^T
// over the context, the ancestors and the node itself, m the greatest score so
// far: one pass over the keys, a tile of 64 at a time. A draft has nodes x group
// queries a key head, which is what a matrix product of 128 rows wants: S = Q K^T
// (both in shared memory) and out = P V (P over its own scores in tensor memory)
// take bf16 operands. What is not bf16 goes in as bf16 parts: fp32 caches and
// queries in three, 24 bits; weights in three, or in two (16 bits, 2^-18 off at
// the most) where cache and result are bf16. Products of parts whose
// places add up to three or more are left out: 2^-24 of the whole. A tile's
// result is added to sums in registers, in rounded fp32: the tensor cores' own
// accumulators cut every addition, which tells after some hundred tiles.
//
// One persistent CTA an SM; all units (tree, key head, block of rows) lie in one
// line of tiles of which each CTA takes an equal share, whatever the lengths.
// Warps by their work, joined by mbarriers: 4 turn scores into weights (a thread
// a row), 8 keep the sums, 2 issue products, 2 bring keys, values and the next
// unit's queries (fp32 caches: 1 brings, 4 split into parts; above 128 channels
// 7 split from registers). A draft of few rows lies in shared memory two or four
// times, each copy taking a share of a tile's keys, so that the weights' threads
// all have work; the copies' sums are joined at a unit's end. Waits have a
// limit, after which the CTA reports, ends, and leaves the join to spoil all of the call's rows.
//
// Measured (queued calls; of the bytes' time at the measured copy rate):
// 24 drafts of 23 after up to 4097 positions, 16 heads of 128, bf16: 129-138 us
// (0.48-0.52): a copy's issue (200 clocks for 16 rows of a page) and what lies
// between a CTA's units (queries, masks, result: 5000 clocks and more).
// 8 drafts of 64 after 32768, 4 key heads of 8, bf16: 575-603 us under the power
// cap, 0.46 PFLOP/s (503 in a short run): the weights' warps, 1650 clocks a
// tile; products 1050. Its keys and values are read once for each 128 rows, four times. With one warp for both kinds of products 1790 and 627 us.
// Two groups of weights' warps that take the tiles in turn: 682 us in a short
// run (96 registers a thread in place of 128, all warps alike: none were moved
// between them); 544 threads in place of 512: 788.
// A chain of 16 after 131071, 2 key heads of 6 of 64, fp32 queries: 53-55 us
// (0.19): three parts of queries and weights, 14 tiles a CTA, then the join, 9.
// 6 fp32 drafts of 37 after up to 2500: 153-156 us, six products a pair of operands
// (48 for a tile's scores, 67 clocks each) and the splitting. A draft of 8
// after 631 positions: 32 us, two tiles a CTA, each step of which is fetched and
// run for the first time. Forms far from their floor, 8 drafts of 24 after 8000, 4
// key heads of 2: heads of 256 bf16 107 us (floor 40), with fp32 queries 249; over
// an fp32 cache 1985 (floor 81; 32 rows a unit, one tile of keys and one of values
// in shared memory, loads by threads in place of TMA); heads of 128 over an fp32
// cache 184 (floor 40), and 186 with bf16 queries, whose two lower parts are
// multiplied although they hold next to nothing.
#pragma once

#include <type_traits>

#include "er_kv_tree.cuh"
#include "er_ptx.cuh"

namespace er {

namespace {

constexpr int kSoftmaxWarps = 4, kSumWarps = 8, kIssueWarp = kSoftmaxWarps + kSumWarps, kLoadWarp = kIssueWarp + 2;

// KP: bf16 parts of a key or value in shared memory (1: as they come from a bf16 cache, 3: of fp32), QP of a query,
// PP of a weight. DP: head_dim padded. ROWS: rows of queries in shared memory (of 128 of a product; the others are
// whatever lies there). TK: keys of a tile. KS, VS: tiles of keys and of values (VD channels of them) in shared memory.
template <int KP_, int QP_, int PP_, int DP_, int ROWS_, int TK_, int KS_, int VS_>
struct TreeShape {
  static constexpr int KP = KP_, QP = QP_, PP = PP_, DP = DP_, ROWS = ROWS_, TK = TK_, KS = KS_, VS = VS_;
  static constexpr int VD = DP < kTreeChannels ? DP : kTreeChannels;
  static constexpr int kKPart = TK * DP * 2, kVPart = TK * VD * 2;  // bytes of one part of a tile
  static constexpr int kKSlot = kKPart * KP, kVSlot = kVPart * KP;
  static constexpr int kQPart = ROWS * DP * 2, kQ = kQPart * QP;
  static_assert(TK == 64, "weights' parts lie 32 columns apart");
  // columns of a tile's scores, then of its weights: two parts over the scores, a third one behind them
  static constexpr int kSP = PP > 2 ? TK * 3 / 2 : TK;
  // tiles of scores (their products are issued ahead, over a unit's end too), and results of a tile, kept while they are read
  static constexpr int SB = 3 * kSP + 2 * VD <= 512 ? 3 : 2, OB = SB * kSP + 2 * VD <= 512 ? 2 : 1;
  // the epilogue's exchange: EC channels of each half at a time, and 4 floats of padding a row
  static constexpr int EC = KP == 1 && QP > 1 && DP == 128 ? 16 : 32, kStagePitch = 2 * EC + 4;
  // fp32 caches, up to 128 channels: RS half tiles as they come, to be split into parts from there
  static constexpr bool kRaw = KP > 1 && DP <= 128;
  static constexpr int RS = kRaw ? 3 : 0, kRawRows = TK / 2, kRawSlot = kRawRows * DP * 4;
  static constexpr int kSmem = kQ + KS * kKSlot + VS * kVSlot + RS * kRawSlot + ROWS * kStagePitch * 4;
  // Warps that fill shared memory. bf16 caches: one that issues the keys' copies, and one the values', which shares the
  // next unit's queries with the scores' products' warp. fp32: one that issues copies and four that split, or seven
  // that split from registers.
  static constexpr int kLoadWarps = KP == 1 ? 2 : kRaw ? 5 : 7, kSplitWarps = KP == 1 ? 0 : kRaw ? 4 : 7;
  static constexpr int kQueryWarps = KP == 1 ? 2 : kSoftmaxWarps;  // of all units but a CTA's first
  // the warps that look at values of drafted keys
  static constexpr int kLookWarps = KP == 1 ? kSoftmaxWarps : kSplitWarps;
  static constexpr int kThreads = (kLoadWarp + kLoadWarps) * 32;
};

// What every wait of a CTA goes by: whether one has given up, and after how many ns one does.
struct TreeWaits {
  volatile int abort;
  unsigned long long limit;
};

template <typename S>
struct TreeShared {
  uint64_t kfull[S::KS], kempty[S::KS], vfull[S::VS], vempty[S::VS], raw[S::VS], looked[S::VS], rfull[S::RS + 1], rempty[S::RS + 1];
  uint64_t qfirst, qfull, qfree, sfull[S::SB], pfull[S::SB], pfree[S::SB], ofull[2], ofree[2], staged, masked, drain[2];
  uint32_t tmem;
  TreeWaits waits;
  TreeRun run;
  TreeScratch scratch;
  TreeWalk walk[S::kThreads / 32];
  int bad_tree[2];
  int16_t parents[2][kMaxNodes];  // of units in turn: a warp may be one ahead of another
  int bad_unit[16];                 // units (numbers + 1) of a bad page, in turn
  uint32_t sees[S::ROWS][9];        // each row's ancestors and itself, a bit a node
  uint32_t vbad[S::VS][S::kLookWarps][S::TK / 32];  // keys of a tile whose value was no number (drafted ones)
  // of tiles in turn: five may be between the weights' warps and the sums'
  float by[8][S::ROWS];             // what a tile's sums so far are multiplied by
  float2 ml[8][S::ROWS];            // maximum and sum of a unit's last tile
};

// Descriptors of operands in shared memory, 128-byte swizzle, eight-row groups 1024 bytes apart: the upper word is
// the same for all, the lower one (address, and for operands whose N is contiguous the distance `lbo` of the next 64
// elements) is put together where the product is issued.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_low(uint32_t addr, uint32_t lbo) { return (addr & 0x3FFFFu) >> 4 | (lbo >> 4) << 16; }

// d (+)= A B, A and B in shared memory, or A in tensor memory; issued by the lane whose `go` is not zero. All lanes
// come here, so the operands may be the warp's.
__device__ __forceinline__ void mma_f16_ss(uint32_t go, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, g;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 g, %6, 0;\n\t"
      "mov.b64 x, {%1, %5};\n\tmov.b64 y, {%2, %5};\n\t"
      "@g tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(kDescHigh), "r"(go)
      : "memory");
}
__device__ __forceinline__ void mma_f16_ts(uint32_t go, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, g;\n\t.reg .b64 y;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 g, %6, 0;\n\t"
      "mov.b64 y, {%2, %5};\n\t"
      "@g tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(kDescHigh), "r"(go)
      : "memory");
}
// arrives on the barrier once the products issued so far are done
__device__ __forceinline__ void commit_on(uint32_t go, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred g;\n\tsetp.ne.b32 g, %1, 0;\n\t"
      "@g tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar),
      "r"(go)
      : "memory");
}
__device__ __forceinline__ uint32_t elected() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r;
}
// a barrier by its address in shared memory
__device__ __forceinline__ bool bar_done(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// a look that does not wait
__device__ __forceinline__ bool bar_is_done(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// the same, asleep until it is done or for 20 us: a warp that waits leaves the issue slots to those that work
__device__ __forceinline__ bool bar_done_asleep(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity), "r"(20000)
      : "memory");
  return ok != 0;
}
static __device__ __noinline__ bool bar_wait_slow(uint32_t bar, uint32_t parity, TreeWaits* waits) {
  if (__all_sync(0xffffffffu, bar_done_asleep(bar, parity))) return true;
  const unsigned long long t0 = globaltimer();
  bool ok = true;
  while (!bar_done_asleep(bar, parity)) {
    if (waits->abort || globaltimer() - t0 > waits->limit) {
      waits->abort = 1;
      ok = false;
      break;
    }
  }
  return __all_sync(0xffffffffu, ok);
}

// A place in a ring of N and how often, modulo 2, it has been gone round.
template <int N>
struct Ring {
  int at = 0;
  uint32_t turn = 0;
  __device__ __forceinline__ void next() {
    if (++at == N) at = 0, turn ^= 1;
  }
};

// bf16 operands, fp32 sums, M = 128; b_mn: B's rows (N) are contiguous, not its K
__device__ __forceinline__ uint32_t idesc_bf16(int n, int b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void async_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void sts16(uint32_t a, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// two floats rounded to bf16, packed, the first one low
__device__ __forceinline__ uint32_t round2(uint64_t v) {
  float x, y;
  unpack2(v, x, y);
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
  return r;
}
// what rounding to `h` has left of v
__device__ __forceinline__ uint64_t rest2(uint64_t v, uint32_t h) {
  return fma2(pack2(__uint_as_float(h << 16), __uint_as_float(h & 0xffff0000u)), pack2(-1.f, -1.f), v);
}

// Eight floats as three bf16 parts, cut, whose sum they are exactly. A part that is zero where the value is not
// takes the least value of its sign: times an infinite key it stays infinite, beside a finite one it vanishes.
__device__ __forceinline__ void split8(const float (&x)[8], uint4 (&out)[3]) {
  uint32_t p[3][8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t b = __float_as_uint(x[j]), tiny = b >> 31 << 15 | 1u;
    const bool finite = (b & 0x7f800000u) != 0x7f800000u;
    p[0][j] = x[j] != x[j] ? 0x7fc0u : b >> 16;
    float rest = finite ? x[j] - __uint_as_float(b & 0xffff0000u) : 0.f;
    p[1][j] = __float_as_uint(rest) >> 16;
    rest -= __uint_as_float(p[1][j] << 16);
    p[2][j] = __float_as_uint(rest) >> 16;
    if (x[j] != 0.f) {
#pragma unroll
      for (int i = 0; i < 3; ++i)
        if ((p[i][j] & 0x7fffu) == 0) p[i][j] = tiny;
    }
  }
#pragma unroll
  for (int i = 0; i < 3; ++i)
    out[i] = make_uint4(p[i][0] | p[i][1] << 16, p[i][2] | p[i][3] << 16, p[i][4] | p[i][5] << 16, p[i][6] | p[i][7] << 16);
}

// Eight finite floats as three bf16 parts, cut, whose sum they are exactly (one that is not finite: parts without a
// number among them).
__device__ __forceinline__ void cut8(const float (&x)[8], uint4 (&out)[3]) {
  uint32_t p[3][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float u = x[2 * j], v = x[2 * j + 1];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      p[i][j] = __byte_perm(__float_as_uint(u), __float_as_uint(v), 0x7632);
      if (i < 2) {
        u -= __uint_as_float(__float_as_uint(u) & 0xffff0000u);
        v -= __uint_as_float(__float_as_uint(v) & 0xffff0000u);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 3; ++i) out[i] = make_uint4(p[i][0], p[i][1], p[i][2], p[i][3]);
}

// Bits of nodes node0 .. node0 + 31 that a row sees; below 0 lies the context, all of which it sees.
__device__ __forceinline__ uint32_t seen_from(const uint32_t* sees, int node0) {
  if (node0 <= -32) return 0xffffffffu;
  if (node0 < 0) return sees[0] << -node0 | ((1u << -node0) - 1);
  const int w = node0 >> 5;
  return __funnelshift_r(w < 8 ? sees[w] : 0u, w < 7 ? sees[w + 1] : 0u, node0 & 31);
}

// (issued by the lane whose `go` is not zero)
__device__ __forceinline__ void tma_box(uint32_t go, uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int slot,
                                        int head, int page) {
  asm volatile(
      "{\n\t.reg .pred g;\n\tsetp.ne.b32 g, %7, 0;\n\t"
      "@g cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], "
      "[%2];\n\t}" ::"r"(dst),
      "l"(map), "r"(bar), "r"(x), "r"(slot), "r"(head), "r"(page), "r"(go)
      : "memory");
}

// Where 16-byte vector c (8 channels) of row r lies in a tile of `rows` rows: 64 channels to a 128-byte line, the
// lines' vectors exchanged by the row (the 128-byte swizzle)
__device__ __forceinline__ uint32_t swizzled(int c, int r, int rows) {
  return (c >> 3) * (rows * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

// the whole warp waits, with a limit; false once any wait of the CTA has given up
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, TreeWaits* waits) {
  if (__all_sync(0xffffffffu, bar_done(bar, parity))) return true;
  return bar_wait_slow(bar, parity, waits);
}

// A unit's queries into shared memory, by `warps` warps of which this is one: eight lanes take a query, which is row
// qi of every replica. Several loads are under way at once, the first ones before the barrier `free` (0: none) says
// that the queries there are used no more.
template <typename S, typename TQ>
__device__ __forceinline__ bool load_queries(const TreeArgs& a, const TreeWalk& w, uint32_t q0, int warp, int warps,
                                             uint32_t free, uint32_t parity, TreeWaits* waits) {
  const int lane = threadIdx.x & 31, d = a.kv.d, R = w.replicas, per = S::ROWS / R, live = w.live;
  // C: 16-byte vectors of bf16 of a lane's query, U queries under way; W: 16-byte words of eight elements
  constexpr int C = S::DP / 64, U = (S::QP == 1 ? 8 : 4) / C > 1 ? (S::QP == 1 ? 8 : 4) / C : 1, W = sizeof(TQ) / 2;
  const int items = (live + 3) / 4, c0 = lane & 7;  // of four queries
  auto ready = [&]() { return free == 0 || bar_wait(free, parity, waits); };
#pragma unroll 1
  for (int i0 = warp; i0 < items; i0 += warps * U) {
    uint4 x[U][C][W];
    const TQ* src[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int qi = (i0 + u * warps) * 4 + lane / 8, q = w.q0 + qi, node = tree_node(a, q);
      src[u] = (const TQ*)a.q + (long long)(w.e.first + node) * a.q_stride +
               (long long)(w.head * a.group + q - node * a.group) * d + c0 * 8;
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int j = 0; j < W; ++j) x[u][c][j] = make_uint4(0, 0, 0, 0);
    }
    auto there = [&](int u, int c) { return (i0 + u * warps) * 4 + lane / 8 < live && (c * 8 + c0) * 8 < d; };
    if (a.q_zero) {
    } else if (a.q_wide) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int c = 0; c < C; ++c)
          if (there(u, c))
#pragma unroll
            for (int j = 0; j < W; ++j) x[u][c][j] = reinterpret_cast<const uint4*>(src[u] + c * 64)[j];
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int c = 0; c < C; ++c)
          if (there(u, c))
#pragma unroll
            for (int j = 0; j < W; ++j) {
              uint32_t h[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if constexpr (sizeof(TQ) == 2)
                  h[e] = (uint32_t)__bfloat16_as_ushort(src[u][c * 64 + 2 * e]) |
                         (uint32_t)__bfloat16_as_ushort(src[u][c * 64 + 2 * e + 1]) << 16;
                else
                  h[e] = __float_as_uint(src[u][c * 64 + 4 * j + e]);
              }
              x[u][c][j] = make_uint4(h[0], h[1], h[2], h[3]);
            }
    }
    if (i0 == warp && !ready()) return false;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int qi = (i0 + u * warps) * 4 + lane / 8;
      if (qi >= live) continue;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        if (c * 8 + c0 >= (d + 15) / 16 * 2) continue;
        uint4 parts[3];
        if constexpr (S::QP == 1) {
          const uint32_t flip = a.q_flip ? 0x80008000u : 0u;
          parts[0] = make_uint4(x[u][c][0].x ^ flip, x[u][c][0].y ^ flip, x[u][c][0].z ^ flip, x[u][c][0].w ^ flip);
        } else {
          float y[8];
#pragma unroll
          for (int j = 0; j < W; ++j) {
            const uint32_t h[4] = {x[u][c][j].x, x[u][c][j].y, x[u][c][j].z, x[u][c][j].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if constexpr (sizeof(TQ) == 2)
                y[2 * e] = __uint_as_float(h[e] << 16), y[2 * e + 1] = __uint_as_float(h[e] & 0xffff0000u);
              else
                y[4 * j + e] = __uint_as_float(h[e]);
            }
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) y[j] = a.q_flip ? -y[j] : y[j];
          split8(y, parts);
        }
        for (int r = 0; r < R; ++r) {
          const uint32_t to = q0 + swizzled(c * 8 + c0, r * per + qi, S::ROWS);
#pragma unroll
          for (int p = 0; p < S::QP; ++p) sts16(to + p * S::kQPart, parts[p]);
        }
      }
    }
  }
  if (warp >= items && !ready()) return false;
  __syncwarp();
  async_fence();
  __syncwarp();
  return true;
}

// The same for later units, one copy for the warps that share it: in place, it costs the weights' warps registers or
// the compiler's order (8 trees of 64 after 32768 604 us in place of 575, but 24 of 23 after 4097 132 in place of 140).
template <typename S, typename TQ>
static __device__ __noinline__ bool next_queries(const TreeArgs& a, const TreeWalk& w, uint32_t q0, int warp, int warps,
                                                 uint32_t free, uint32_t parity, TreeWaits* waits) {
  return load_queries<S, TQ>(a, w, q0, warp, warps, free, parity, waits);
}

template <typename S, typename TC, typename TQ>
__global__ void __launch_bounds__(S::kThreads, 1)
    kv_tree_kernel(const __grid_constant__ TreeArgs a, const __grid_constant__ CUtensorMap kmap,
                   const __grid_constant__ CUtensorMap vmap) {
  extern __shared__ unsigned char raw[];
  __shared__ TreeShared<S> s;
  constexpr int TK = S::TK, KS = S::KS, VS = S::VS, SB = S::SB, OB = S::OB;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = a.kv.d;
  const uint32_t base = (smem_u32(raw) + 1023) & ~1023u;  // swizzled tiles repeat every 1024 bytes
  // the queries first: products read 128 rows from there, whatever lies behind S::ROWS
  const uint32_t q0 = base, k0 = q0 + S::kQ, v0 = k0 + KS * S::kKSlot, raw0 = v0 + VS * S::kVSlot;
  float* stage = reinterpret_cast<float*>(raw + (raw0 + S::RS * S::kRawSlot - smem_u32(raw)));

  if (threadIdx.x == 0) {
    for (int i = 0; i < KS; ++i) mbar_init(&s.kfull[i], S::KP == 1 ? 1 : S::kSplitWarps), mbar_init(&s.kempty[i], 1);
    for (int i = 0; i < VS; ++i) {
      mbar_init(&s.vfull[i], S::kLookWarps);
      mbar_init(&s.vempty[i], 1);
      mbar_init(&s.raw[i], 1);
      mbar_init(&s.looked[i], S::kLookWarps);
    }
    for (int i = 0; i < S::RS; ++i) mbar_init(&s.rfull[i], 1), mbar_init(&s.rempty[i], S::kSplitWarps);
    mbar_init(&s.qfirst, kIssueWarp);
    mbar_init(&s.qfull, S::kQueryWarps);
    mbar_init(&s.qfree, 1);
    for (int i = 0; i < SB; ++i) mbar_init(&s.sfull[i], 1), mbar_init(&s.pfull[i], kSoftmaxWarps), mbar_init(&s.pfree[i], 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.ofull[i], 1);
      mbar_init(&s.ofree[i], kSumWarps);
    }
    mbar_init(&s.staged, kSumWarps);
    mbar_init(&s.masked, kSoftmaxWarps);
    for (int i = 0; i < 2; ++i) mbar_init(&s.drain[i], 1);
    s.waits.abort = 0, s.waits.limit = a.wait_ns;
    s.bad_tree[0] = s.bad_tree[1] = 0;
    for (int i = 0; i < 16; ++i) s.bad_unit[i] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kIssueWarp) tmem_alloc<1>(&s.tmem, 512);
  kv_enter();
  tree_run(a, s.run, s.scratch);  // all threads; ends with a barrier
  tc_fence_after();
  const uint32_t tmem = s.tmem;
  auto wait = [&](const uint64_t& b, uint32_t parity) { return bar_wait(smem_u32(&b), parity, &s.waits); };
  auto arrive = [&](const uint64_t& b) {  // the warp's one arrival, after all its lanes
    __syncwarp();
    if (lane == 0) bar_arrive(smem_u32(&b));
  };
  const TreeWalk& w = s.walk[warp];
  auto next = [&](bool first) { return tree_next(a, s.run, &s.walk[warp], first, S::ROWS / 32); };
  if (warp < kIssueWarp && next(true)) {  // the first unit's queries by the warps that have nothing to do yet
    load_queries<S, TQ>(a, w, q0, warp, kIssueWarp, 0, 0, &s.waits);
    arrive(s.qfirst);
  }

  if (warp < kSoftmaxWarps) {
    // ---- weights: a thread a row, of one replica's share of the tile's keys
    int it = 0, masks = 0, unit = 0, looks = 0;
    Ring<SB> sp_ring;
    Ring<VS> v_ring;
#pragma unroll 1
    for (bool go = next(true); go && !s.waits.abort; go = next(false), ++unit) {
      if (S::KP > 1 && unit > 0) {  // the first one's are on their way
        if (!load_queries<S, TQ>(a, w, q0, warp, kSoftmaxWarps, smem_u32(&s.qfree), (unit - 1) & 1, &s.waits)) break;
        arrive(s.qfull);
      }
      const int R = w.replicas, per = S::ROWS / R, row = threadIdx.x, len = w.e.len, lo = w.lo, hi = w.hi;
      const int qi = row % per, slice = row < S::ROWS ? row / per : 0;
      const bool mine = row < S::ROWS && qi < w.live, live = __any_sync(0xffffffffu, mine);
      uint32_t* sees = s.sees[row < S::ROWS ? row : 0];
      float m = -INFINITY, l = 0.f;
      // the rows' masks, where this CTA meets drafted keys
      bool masked = false;
      auto mask = [&]() {
        for (int i = threadIdx.x; i < w.e.nodes; i += kSoftmaxWarps * 32) {
          int p = a.parents[w.e.first + i];
          if (p < -1 || p >= i) {
            kv_report(a.status, ER_KV_BAD_TREE);
            s.bad_tree[masks & 1] = masks + 1;  // of this unit
            p = -1;
          }
          s.parents[masks & 1][i] = (int16_t)p;
        }
        arrive(s.masked);
        if (!wait(s.masked, masks & 1)) return false;
        if (row < S::ROWS)
          for (int i = 0; i < 9; ++i) sees[i] = 0;
        if (mine)
          for (int p = tree_node(a, w.q0 + qi); p >= 0; p = s.parents[masks & 1][p]) sees[p >> 5] |= 1u << (p & 31);
        if (s.bad_tree[masks & 1] == masks + 1) l = __int_as_float(0x7fc00000);
        ++masks;
        __syncwarp();
        return masked = true;
      };
      // values of drafted keys, and of places behind the last one, in shared memory: zero where they are no numbers,
      // for the rows that do not see them, and marked for those that do
      auto look = [&](int t, int slot) {
        const uint32_t to = v0 + slot * S::kVSlot;
        const int vv = (min(S::VD, d - w.ch0) + 15) / 16 * 2, r0 = len - t * TK, r9 = len + w.e.nodes - t * TK;
        uint32_t marks[TK / 32] = {};
#pragma unroll
        for (int h = 0; h < S::VD / 64; ++h) {
          const int c = h * 8 + (lane & 7);
          uint4 v[TK / 16];
#pragma unroll
          for (int j = 0; j < TK / 16; ++j) v[j] = lds16(to + swizzled(c, j * 16 + warp * 4 + lane / 8, TK));
#pragma unroll
          for (int j = 0; j < TK / 16; ++j) {
            const int r = j * 16 + warp * 4 + lane / 8;
            const uint32_t e[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
            uint32_t bad = 0;  // whether an exponent is all ones
#pragma unroll
            for (int i = 0; i < 4; ++i) bad |= ((e[i] & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
            if (r < r0 || c >= vv || !(bad || r >= r9)) continue;
            sts16(to + swizzled(c, r, TK), make_uint4(0, 0, 0, 0));
            if (bad) marks[j / 2] |= 1u << (r & 31);
          }
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < TK / 32; ++i) {
          marks[i] = __reduce_or_sync(0xffffffffu, marks[i]);
          if (lane == 0) s.vbad[slot][warp][i] = marks[i];
        }
        async_fence();
        arrive(s.vfull[slot]);
        arrive(s.looked[slot]);
      };
      const uint32_t sp0 = tmem + ((uint32_t)(warp * 32) << 16);
      // N scores of this row into x: those of the keys from key on of tile t, -inf where the row does not see them
      auto scores = [&](auto& x, int t, int key) {
        constexpr int N = sizeof(x) / 4;
        const uint32_t sp = sp0 + sp_ring.at * S::kSP + key;
        if constexpr (N == 16) {
          tmem_ld16(sp, x);
        } else {
          tmem_ld32(sp, x);
          if constexpr (N == 64) tmem_ld32(sp + 32, x + 32);
        }
        tmem_wait_ld();
        const int node0 = t * TK + key - len;
        if (node0 + N > 0) {  // drafted keys, or none
          uint32_t spoils = 0;
#pragma unroll
          for (int c = 0; c < N; c += 32) {
            const uint32_t see = seen_from(sees, node0 + c);
#pragma unroll
            for (int j = c; j < N && j < c + 32; ++j)
              if (!(see >> (j - c) & 1)) x[j] = 0xff800000u;
            uint32_t vb = 0;
            for (int i = 0; i < S::kLookWarps; ++i) vb |= s.vbad[v_ring.at][i][(key + c) >> 5] >> ((key + c) & 31);
            spoils |= vb & see & (N < 32 ? (1u << (N & 31)) - 1 : 0xffffffffu);
          }
          if (spoils) l = __int_as_float(0x7fc00000);
        }
      };
      // the weights of N scores, as they are multiplied: in parts, from column c on; their sum
      auto weights = [&](auto& x, float shift, int c) {
        constexpr int N = sizeof(x) / 4;
        const uint32_t sp = sp0 + sp_ring.at * S::kSP + c;
        const uint64_t scale = pack2(a.scale, a.scale), by = pack2(shift, shift);
        uint64_t sum = 0;  // of even and of odd keys
#pragma unroll
        for (int i = 0; i < N / 2; i += 8) {
          uint64_t p[8];
          uint32_t y[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            float u, v;
            unpack2(fma2(pack2(__uint_as_float(x[2 * (i + j)]), __uint_as_float(x[2 * (i + j) + 1])), scale, by), u, v);
            p[j] = pack2(ex2(u), ex2(v));
            sum = add2(sum, p[j]);
          }
#pragma unroll
          for (int part = 0; part < S::PP; ++part) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              y[j] = round2(p[j]);
              if (part + 1 < S::PP) p[j] = rest2(p[j], y[j]);
            }
            tmem_st8(sp + part * 32 + i, y);
          }
        }
        float even, odd;
        unpack2(sum, even, odd);
        return even + odd;
      };
      // what the sums so far are multiplied by, once the greatest score is `top`, and the exponents' shift
      auto rise = [&](float top, float* shift) {
        const float ref = top == -INFINITY ? 0.f : top;
        *shift = __fmul_rn(-ref, a.scale);
        // by the difference of the two shifts as they are, rounded: 1 where the greatest score stays. (With a product
        // that is not rounded it is 1 and what the shift's rounding took, once a tile: 1e-5 of a result of 32768 keys.)
        const float by = ex2(__fadd_rn(__fmul_rn(m, a.scale), *shift));
        m = top;
        if (row < S::ROWS) s.by[it & 7][row] = by;
        __syncwarp();
        return by;
      };
      auto tile = [&](auto replicas, int t) {
        constexpr int RR = decltype(replicas)::value, KPT = TK / RR;
        uint32_t x[KPT];
        float top = m, shift;
        const int key = slice * KPT;
        scores(x, t, key);
#pragma unroll
        for (int j = 0; j < KPT; ++j) top = fmaxf(top, __uint_as_float(x[j]));
        const float by = rise(top, &shift);
        l = l * by + weights(x, shift, key / 2);
        // the other keys are other replicas'
        const uint32_t zero[8] = {};
        const uint32_t sp = sp0 + sp_ring.at * S::kSP;
#pragma unroll
        for (int c = KPT / 2; c < TK / 2; c += 8) {
          const int at = (key / 2 + c) & (TK / 2 - 1);
#pragma unroll
          for (int part = 0; part < S::PP; ++part) tmem_st8(sp + part * 32 + at, zero);
        }
      };
      bool ok = true;
#pragma unroll 1
      for (int t = lo; t < hi; ++t, ++it, sp_ring.next(), v_ring.next()) {
        if (!(ok = wait(s.sfull[sp_ring.at], sp_ring.turn))) break;
        if ((t + 1) * TK > len) {  // its values are looked at first
          const uint32_t turn = looks >> v_ring.at & 1;
          if (!masked && !(ok = mask())) break;
          if (S::KP == 1) {
            if (!(ok = wait(s.raw[v_ring.at], turn))) break;
            look(t, v_ring.at);
          }
          if (!(ok = wait(s.looked[v_ring.at], turn))) break;
          looks ^= 1 << v_ring.at;
        }
        tc_fence_after();
        if (live) {
          if (R == 1)
            tile(std::integral_constant<int, 1>{}, t);
          else if (R == 2)
            tile(std::integral_constant<int, 2>{}, t);
          else
            tile(std::integral_constant<int, 4>{}, t);
          tmem_wait_st();
        }
        if (t + 1 == hi && row < S::ROWS) {
          if (s.bad_unit[unit & 15] == unit + 1) l = __int_as_float(0x7fc00000);
          s.ml[it & 7][row] = make_float2(m == -INFINITY ? m : m * a.scale, l);
        }
        tc_fence_before();
        arrive(s.pfull[sp_ring.at]);
      }
      if (!ok) break;
    }
  } else if (warp < kIssueWarp) {
    // ---- sums: a thread a row, of half of the channels
    constexpr int CH = S::VD / 2, EC = S::EC, kStagePitch = S::kStagePitch;
    const int row = (warp & 3) * 32 + lane, half = (warp - kSoftmaxWarps) >> 2, id = threadIdx.x - kSoftmaxWarps * 32;
    int it = 0;
    Ring<OB> o_ring;
    uint32_t stages = 0;
    if (id == 0) a.cut[blockIdx.x].live = 0;
#pragma unroll 1
    for (bool go = next(true); go && !s.waits.abort; go = next(false)) {
      uint64_t o[CH / 2];  // two channels each
#pragma unroll
      for (int c = 0; c < CH / 2; ++c) o[c] = 0;
      const int R = w.replicas, per = S::ROWS / R, vd = min(S::VD, d - w.ch0);
      const bool there = row < S::ROWS, live = __any_sync(0xffffffffu, there && row % per < w.live);
      bool ok = true;
      float2 ml = make_float2(0.f, 0.f);
      const int hi = w.hi;
#pragma unroll 1
      for (int t = w.lo; t < hi; ++t, ++it, o_ring.next()) {
        const int ob = o_ring.at;
        if (!(ok = wait(s.ofull[ob], o_ring.turn))) break;  // after the tile's weights, so `by` and `ml` are there
        tc_fence_after();
        if (live) {
          const float by1 = there ? s.by[it & 7][row] : 0.f;
          const uint64_t by = pack2(by1, by1);
          const uint32_t at = tmem + ((uint32_t)((warp & 3) * 32) << 16) + SB * S::kSP + ob * S::VD + half * CH;
          constexpr int N = S::KP > 1 ? 16 : 32;  // registers
#pragma unroll
          for (int c = 0; c < CH; c += N) {
            uint32_t x[N];
            if constexpr (N == 32)
              tmem_ld32(at + c, x);
            else
              tmem_ld16(at + c, x);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < N; j += 2)
              o[(c + j) / 2] = fma2(o[(c + j) / 2], by, pack2(__uint_as_float(x[j]), __uint_as_float(x[j + 1])));
          }
        }
        if (t + 1 == hi && there) ml = s.ml[it & 7][row];
        tc_fence_before();
        arrive(s.ofree[ob]);
      }
      if (!ok) break;
      // the replicas' rows joined, by way of shared memory
      const bool whole = w.lo == 0 && w.hi == w.u.tiles, begins = w.lo == 0;
      if (!whole && begins && id == 0)
        a.cut[blockIdx.x] = TreeCut{w.e.first, w.head, w.q0, w.live, w.u.tiles, w.ch0, w.pos, s.run.total};
      const long long piece = (long long)blockIdx.x * 2 + begins;
#pragma unroll
      for (int c0 = 0; c0 < CH; c0 += EC) {
        if (there) {
          float* mine = stage + row * kStagePitch + half * EC;
#pragma unroll
          for (int j = 0; j < EC; j += 4)
            *reinterpret_cast<ulonglong2*>(mine + j) = make_ulonglong2(o[(c0 + j) / 2], o[(c0 + j) / 2 + 1]);
          if (c0 == 0 && half == 0) *reinterpret_cast<float2*>(stage + row * kStagePitch + 2 * EC) = ml;
        }
        arrive(s.staged);
        if (!(ok = wait(s.staged, stages))) break;
        stages ^= 1;
        for (int i = id; i < w.live * (EC / 2); i += kSumWarps * 32) {
          const int qi = i / (EC / 2), hh = i / (EC / 4) & 1, v = i % (EC / 4), ch = hh * CH + c0 + v * 4;
          if (ch >= vd) continue;
          float2 p[4];
          float4 x[4];
          float top = -INFINITY, sum = 0.f;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            p[r] = make_float2(-INFINITY, 0.f);
            x[r] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < R) {
              const float* at = stage + (r * per + qi) * kStagePitch;
              p[r] = *reinterpret_cast<const float2*>(at + 2 * EC);
              x[r] = *reinterpret_cast<const float4*>(at + hh * EC + v * 4);
            }
            top = fmaxf(top, p[r].x);
          }
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float by = piece_weight(p[r].x, top);
            sum = fmaf(p[r].y, by, sum);  // a spoilt row's sum is NaN
            fma4(acc, x[r], by);
          }
          if (whole) {
            const int q = w.q0 + qi, node = tree_node(a, q), g = q - node * a.group;
            const long long at = (long long)(w.e.first + node) * a.heads + w.head * a.group + g;
            kv_store4((TQ*)a.out + at * d + w.ch0 + ch, acc, sum);
          } else {
            *reinterpret_cast<float4*>(a.part_o + (piece * a.piece_rows + qi) * S::VD + ch) = acc;
            if (ch == 0) *reinterpret_cast<float2*>(a.part_ml + (piece * a.piece_rows + qi) * 2) = make_float2(top, sum);
          }
        }
        arrive(s.staged);
        if (!(ok = wait(s.staged, stages))) break;
        stages ^= 1;
      }
      if (!ok) break;
    }
    if (a.stall) wait(s.drain[0], 0);  // which nothing completes
  } else if (warp <= kIssueWarp + 1) {
    // ---- products: a warp's for scores, another's for results, so that neither waits for what the other needs
    constexpr bool kThree = S::KP > 1;  // products of parts i and j: those with i + j > 2 are under 2^-24 of the whole
    const uint32_t one = elected();
    Ring<SB> ring;  // of tiles of scores or weights
    int tiles = 0;
    bool ok = true;
    // Descriptors are put together where they are used, from words the compiler cannot know before, so that none lives
    // over a call (bar_wait_slow, tree_next, next_queries): over those live 32-bit addresses, rings and counts only.
    // The small products first.
    if (warp == kIssueWarp) {
      const int ksteps = (d + 15) / 16;
      const uint32_t is = idesc_bf16(TK, 0);
      int unit = 0;
      Ring<KS> k_ring, last_k;
#pragma unroll 1
      for (bool go = next(true); go && ok; go = next(false), ++unit) {
        if (S::KP == 1 && unit > 0) {  // half of its queries, which nothing goes on without
          if (!(ok = next_queries<S, TQ>(a, w, q0, 1, 2, smem_u32(&s.qfree), (unit - 1) & 1, &s.waits))) break;
          arrive(s.qfull);
        }
        if (!(ok = unit ? wait(s.qfull, (unit - 1) & 1) : wait(s.qfirst, 0))) break;
        const int hi = w.hi;
#pragma unroll 1
        for (int t = w.lo; t < hi; ++t, ++tiles, ring.next(), k_ring.next()) {
          if (tiles >= SB && !(ok = wait(s.pfree[ring.at], ring.turn ^ 1))) break;
          if (!(ok = wait(s.kfull[k_ring.at], k_ring.turn))) break;
          tc_fence_after();
          uint32_t kd = desc_low(k0 + k_ring.at * S::kKSlot, 16), qd = desc_low(q0, 16);
          uint32_t to = tmem + ring.at * S::kSP, id = is;
          asm volatile("" : "+r"(kd), "+r"(qd), "+r"(to), "+r"(id));
#pragma unroll
          for (int qp = S::QP - 1; qp >= 0; --qp)
#pragma unroll
            for (int kp = S::KP - 1; kp >= 0; --kp) {
              if (kThree && qp + kp > 2) continue;
#pragma unroll
              for (int k = 0; k < S::DP / 16; ++k)
                mma_f16_ss(k < ksteps ? one : 0u, to, qd + ((qp * S::kQPart + (k >> 2) * (S::ROWS * 128) + (k & 3) * 32) >> 4),
                           kd + ((kp * S::kKPart + (k >> 2) * (TK * 128) + (k & 3) * 32) >> 4), id,
                           !(qp == S::QP - 1 && kp == (kThree ? 2 - qp : 0) && k == 0));
            }
          commit_on(one, smem_u32(&s.sfull[ring.at]));
          commit_on(one, smem_u32(&s.kempty[k_ring.at]));
          if (t + 1 == hi) commit_on(one, smem_u32(&s.qfree));
          last_k = k_ring;
        }
        if (!ok) break;
      }
      // no arrival is under way when the CTA ends
      if (ok && unit > 0) ok = wait(s.kempty[last_k.at], last_k.turn) && wait(s.qfree, (unit - 1) & 1);
    } else {
      Ring<OB> o_ring;
      Ring<VS> v_ring, last_v;
      Ring<SB> last;
#pragma unroll 1
      for (bool go = next(true); go && ok; go = next(false)) {
        const uint32_t io = idesc_bf16((min(S::VD, d - w.ch0) + 15) / 16 * 16, 1);
        const int hi = w.hi;
#pragma unroll 1
        for (int t = w.lo; t < hi; ++t, ++tiles, ring.next(), o_ring.next(), v_ring.next()) {
          const int b = o_ring.at;
          if (!(ok = wait(s.vfull[v_ring.at], v_ring.turn))) break;
          if (tiles >= OB && !(ok = wait(s.ofree[b], o_ring.turn ^ 1))) break;
          if (!(ok = wait(s.pfull[ring.at], ring.turn))) break;
          tc_fence_after();
          uint32_t v = desc_low(v0 + v_ring.at * S::kVSlot, TK * 128);
          uint32_t to = tmem + SB * S::kSP + b * S::VD, p = tmem + ring.at * S::kSP, id = io;
          asm volatile("" : "+r"(v), "+r"(to), "+r"(p), "+r"(id));
#pragma unroll
          for (int pp = S::PP - 1; pp >= 0; --pp)
#pragma unroll
            for (int kp = S::KP - 1; kp >= 0; --kp) {
              if (kThree && pp + kp > 2) continue;
#pragma unroll
              for (int k = 0; k < TK / 16; ++k)
                mma_f16_ts(one, to, p + pp * 32 + k * 8, v + ((kp * S::kVPart + k * 2048) >> 4), id,
                           !(pp == S::PP - 1 && kp == (kThree ? 2 - pp : 0) && k == 0));
            }
          commit_on(one, smem_u32(&s.ofull[b]));
          commit_on(one, smem_u32(&s.pfree[ring.at]));
          commit_on(one, smem_u32(&s.vempty[v_ring.at]));
          last = ring;
          last_v = v_ring;
        }
        if (!ok) break;
      }
      if (ok && tiles > 0) ok = wait(s.pfree[last.at], last.turn) && wait(s.vempty[last_v.at], last_v.turn);
    }
    if (!ok) {  // the products under way end before their memory goes
      uint64_t* drain = &s.drain[warp - kIssueWarp];
      commit_on(one, smem_u32(drain));
      mbar_drain(drain, 0, kDefaultWaitNs);
    }
    __syncwarp();
  } else if (S::kRaw && warp == kLoadWarp) {
    // ---- copies of fp32 keys and values, half a tile each, in the order in which they are split: the next tile's
    // keys before a tile's values
    const int rows = a.box_rows, each = S::kRawRows / rows;
    const uint32_t one = elected();
    Ring<S::kRaw ? S::RS : 1> ring;
    int unit = 0, item = 0;
    bool ok = true;
#pragma unroll 1
    for (bool go = next(true); go && ok && !s.waits.abort; go = next(false), ++unit) {
      const int32_t* pages = a.kv.pages_of(w.e.seq);
      const int keys = w.e.len + w.e.nodes, hi = w.hi, head = w.head;
      auto page_of = [&](int t, int i) {  // of box i; behind the last key none
        const int key = t * TK + i * rows;
        return t < hi && i < 2 * each && key < keys ? pages[a.kv.ordinal(key)] : a.kv.num_pages;
      };
      auto checked = [&](int page, int t, int i) {
        if (page >= 0 && page < a.kv.num_pages) return page;
        if (t < hi && i < 2 * each && t * TK + i * rows < keys) {
          kv_report(a.status, ER_KV_BAD_PAGE);
          s.bad_unit[unit & 15] = unit + 1;
        }
        return a.kv.num_pages;  // outside the pool: zeros
      };
      auto copy = [&](int t, const int (&page)[2], const CUtensorMap* map) {
#pragma unroll 1
        for (int h = 0; h < 2; ++h, ++item, ring.next()) {
          if (item >= S::RS && !(ok = wait(s.rempty[ring.at], ring.turn ^ 1))) return;
          const uint32_t bar = smem_u32(&s.rfull[ring.at]);
          asm volatile(
              "{\n\t.reg .pred g;\n\tsetp.ne.b32 g, %2, 0;\n\t"
              "@g mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}" ::"r"(bar),
              "r"(S::kRawSlot), "r"(one)
              : "memory");
          uint32_t to = raw0 + ring.at * S::kRawSlot;
          int at = a.kv.slot(t * TK + h * S::kRawRows);
#pragma unroll 1
          for (int b = 0; b < each; ++b, to += rows * S::DP * 4) {
            const int i = h * each + b, pg = __shfl_sync(0xffffffffu, i < 32 ? page[0] : page[1], i & 31);
            tma_box(one, to, map, bar, 0, at, head, pg);
            at = at + rows == a.kv.page_size ? 0 : at + rows;
          }
        }
      };
      int now[2], then[2] = {page_of(w.lo, lane), page_of(w.lo, lane + 32)};
#pragma unroll
      for (int j = 0; j < 2; ++j) now[j] = checked(then[j], w.lo, lane + 32 * j), then[j] = page_of(w.lo + 1, lane + 32 * j);
      copy(w.lo, now, &kmap);
#pragma unroll 1
      for (int t = w.lo; t < hi && ok; ++t) {
#pragma unroll
        for (int j = 0; j < 2; ++j) then[j] = checked(then[j], t + 1, lane + 32 * j);
        __syncwarp();
        if (t + 1 < hi) copy(t + 1, then, &kmap);
        if (ok) copy(t, now, &vmap);
#pragma unroll
        for (int j = 0; j < 2; ++j) now[j] = then[j], then[j] = page_of(t + 2, lane + 32 * j);
      }
    }
  } else if constexpr (S::KP == 1) {
    // ---- copies of keys, or of values and a unit's queries: boxes of as many positions as lie in one page
    const bool values = warp == kLoadWarp + 1;
    const int rows = a.box_rows, boxes = TK / rows, box_shift = __ffs(boxes) - 1, ring = values ? VS : KS;
    const CUtensorMap* map = values ? &vmap : &kmap;
    const uint32_t one = elected(), slots0 = values ? v0 : k0, slot_bytes = values ? S::kVSlot : S::kKSlot;
    int unit = 0, it = 0, at_slot = 0;
    uint32_t turn = 0;
    bool ok = true;
#pragma unroll 1
    for (bool go = next(true); go && ok && !s.waits.abort; go = next(false), ++unit) {
      if (values && unit > 0) {  // its queries first; the first unit's are on their way
        if (!(ok = next_queries<S, TQ>(a, w, q0, 0, 2, smem_u32(&s.qfree), (unit - 1) & 1, &s.waits))) break;
        arrive(s.qfull);
      }
      const int32_t* pages = a.kv.pages_of(w.e.seq);
      const int len = w.e.len, keys = len + w.e.nodes, x0 = values ? w.ch0 : 0;
      const int chunks = ((values ? min(S::VD, d - w.ch0) : d) + 63) / 64;
      // the pages of the unit's boxes, one after another: the lanes hold 32 of them and the 32 behind those
      const int hi = w.hi, lo = w.lo, head = w.head;
      auto pages_from = [&](int first) {
        const int n = first + lane, key = (lo + (n >> box_shift)) * TK + (n & (boxes - 1)) * rows;
        if (lo + (n >> box_shift) >= hi || key >= keys) return a.kv.num_pages;
        const int page = pages[a.kv.ordinal(key)];
        if (page >= 0 && page < a.kv.num_pages) return page;
        kv_report(a.status, ER_KV_BAD_PAGE);
        s.bad_unit[unit & 15] = unit + 1;
        return a.kv.num_pages;  // outside the pool: zeros
      };
      int now = pages_from(0), then = pages_from(32), n = 0, first = 0;
#pragma unroll 1
      for (int t = lo; t < hi; ++t, ++it) {
        __syncwarp();
        if (it >= ring && !(ok = wait(values ? s.vempty[at_slot] : s.kempty[at_slot], turn ^ 1))) break;
        // values of a tile with drafted keys are looked at before they count
        const bool whole = !values || (t + 1) * TK <= len;
        const uint32_t bar = smem_u32(!values ? &s.kfull[at_slot] : whole ? &s.vfull[at_slot] : &s.raw[at_slot]);
        if (values && whole && one)
          for (int i = 1; i < S::kLookWarps; ++i) bar_arrive(bar);
        __syncwarp();
        asm volatile(
            "{\n\t.reg .pred g;\n\tsetp.ne.b32 g, %2, 0;\n\t"
            "@g mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}" ::"r"(bar),
            "r"(chunks * TK * 128), "r"(one)
            : "memory");
        uint32_t to = slots0 + at_slot * slot_bytes;
        int at = a.kv.slot(t * TK);
        auto box = [&](int pg) {
#pragma unroll
          for (int c = 0; c < S::DP / 64; ++c)
            if (c < chunks) tma_box(one, to + c * (TK * 128), map, bar, x0 + c * 64, at, head, pg);
          to += rows * 128;
          at = at + rows == a.kv.page_size ? 0 : at + rows;
        };
        if (boxes <= 4) {  // their pages first: each exchange would be waited for
          int pg[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) pg[i] = __shfl_sync(0xffffffffu, now, n + i);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (i < boxes) box(pg[i]);
          n += boxes;
        } else {
#pragma unroll 1
          for (int i = 0; i < boxes; ++i, ++n) {
            if (n == 32) n = 0, now = then, first += 32, then = pages_from(first + 32);
            box(__shfl_sync(0xffffffffu, now, n));
          }
        }
        if (n == 32) n = 0, now = then, first += 32, then = pages_from(first + 32);
        if (++at_slot == ring) at_slot = 0, turn ^= 1;
      }
    }
  } else {
    // ---- keys and values split into parts (fp32 caches)
    const int loader = warp - (kLoadWarp + S::kLoadWarps - S::kSplitWarps);
    int unit = 0, it = 0, k_item = 0;
    Ring<KS> k_ring;
    Ring<VS> v_ring;
    Ring<S::kRaw ? S::RS : 1> r_ring;
    bool ok = true;
    auto signal = [&](const uint64_t& b) {
      async_fence();
      arrive(b);
    };
#pragma unroll 1
    for (bool go = next(true); go && ok && !s.waits.abort; go = next(false), ++unit) {
      const int keys = w.e.len + w.e.nodes;
      if constexpr (S::kRaw) {
        const int len = w.e.len, hi = w.hi;
        constexpr int ITEMS = (S::kRawRows / 4 * (S::DP / 64) + S::kSplitWarps - 1) / S::kSplitWarps;  // four rows, 64 channels
        auto split = [&](int t, const uint64_t& full, uint32_t to, int part, bool look, int slot) {
          uint32_t marks[TK / 32] = {};
#pragma unroll 1
          for (int h = 0; h < 2; ++h, r_ring.next()) {
            if (!(ok = wait(s.rfull[r_ring.at], r_ring.turn))) return;
            const uint32_t from = raw0 + r_ring.at * S::kRawSlot;
            uint4 u[ITEMS], v[ITEMS];
            // eight lanes read 256 bytes of a row: four of them their second 16 bytes first, for the banks
            const uint32_t swap = (lane & 4) * 4;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
              const int n = loader + i * S::kSplitWarps, r = n / (S::DP / 64) * 4 + lane / 8, c = n % (S::DP / 64) * 8 + (lane & 7);
              if (r >= S::kRawRows) continue;
              u[i] = lds16(from + r * (S::DP * 4) + c * 32 + swap);
              v[i] = lds16(from + r * (S::DP * 4) + c * 32 + (swap ^ 16));
            }
            arrive(s.rempty[r_ring.at]);
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
              const int n = loader + i * S::kSplitWarps, r0 = n / (S::DP / 64) * 4 + lane / 8, c = n % (S::DP / 64) * 8 + (lane & 7);
              const int r = h * S::kRawRows + r0;
              if (r0 >= S::kRawRows) continue;
              const uint4 x = swap ? v[i] : u[i], z = swap ? u[i] : v[i];
              float y[8] = {__uint_as_float(x.x), __uint_as_float(x.y), __uint_as_float(x.z), __uint_as_float(x.w),
                            __uint_as_float(z.x), __uint_as_float(z.y), __uint_as_float(z.z), __uint_as_float(z.w)};
              if (look && t * TK + r >= len) {  // values of drafted tokens, and what lies behind the last one
                bool bad = false;
#pragma unroll
                for (int j = 0; j < 8; ++j) bad |= !(fabsf(y[j]) < INFINITY);
                if (bad || t * TK + r >= keys) {
#pragma unroll
                  for (int j = 0; j < 8; ++j) y[j] = 0.f;
                }
#pragma unroll
                for (int j = 0; j < TK / 32; ++j)
                  if (bad && r >> 5 == j) marks[j] |= 1u << (r & 31);
              }
              uint4 parts[3];
              cut8(y, parts);
              const uint32_t dst = to + swizzled(c, r, TK);
#pragma unroll
              for (int j = 0; j < 3; ++j) sts16(dst + j * part, parts[j]);
            }
          }
          __syncwarp();
          if (look) {
#pragma unroll
            for (int i = 0; i < TK / 32; ++i) {
              marks[i] = __reduce_or_sync(0xffffffffu, marks[i]);
              if (lane == 0) s.vbad[slot][loader][i] = marks[i];
            }
          }
          signal(full);
          if (look) arrive(s.looked[slot]);
        };
        auto keys_of = [&](int t) {
          if (k_item >= KS && !(ok = wait(s.kempty[k_ring.at], k_ring.turn ^ 1))) return;
          split(t, s.kfull[k_ring.at], k0 + k_ring.at * S::kKSlot, S::kKPart, false, 0);
          k_ring.next();
          ++k_item;
        };
        auto values_of = [&](int t) {
          if (it >= VS && !(ok = wait(s.vempty[v_ring.at], v_ring.turn ^ 1))) return;
          split(t, s.vfull[v_ring.at], v0 + v_ring.at * S::kVSlot, S::kVPart, (t + 1) * TK > len, v_ring.at);
          v_ring.next();
          ++it;
        };
        keys_of(w.lo);
#pragma unroll 1
        for (int t = w.lo; t < hi && ok; ++t) {
          if (t + 1 < hi) keys_of(t + 1);
          if (ok) values_of(t);
        }
      } else {
        // a step: up to 128 channels of the rows in groups of four, eight lanes a row and 64 channels
        constexpr int GROUPS = (TK / 4 + S::kSplitWarps - 1) / S::kSplitWarps;
        const int32_t* pages = a.kv.pages_of(w.e.seq);
        const int hi = w.hi, len = w.e.len;
        auto row_of = [&](int i) { return (loader + i * S::kSplitWarps) * 4; };
        const int own = row_of(lane >> 2) + (lane & 3);  // the row that this lane looks up
        const bool looks_up = lane < GROUPS * 4 && own < TK;
        auto page_of = [&](int t) {
          const int key = t * TK + own;
          return t < hi && looks_up && key < keys ? pages[a.kv.ordinal(key)] : -1;
        };
        auto place_of = [&](int t, int page) -> long long {  // in the pools; -1: none, or a bad page
          const int key = t * TK + own;
          if (!looks_up || key >= keys) return -1;
          if (page < 0 || page >= a.kv.num_pages) {
            kv_report(a.status, ER_KV_BAD_PAGE);
            s.bad_unit[unit & 15] = unit + 1;
            return -1;
          }
          return page * a.kv.page_stride + w.head * a.kv.head_stride + a.kv.slot(key) * a.kv.slot_stride;
        };
        float4 x[2][GROUPS][2];
        long long off = place_of(w.lo, page_of(w.lo));
        int page = page_of(w.lo + 1);
        const int widths[2] = {d, min(S::VD, d - w.ch0)}, ch0 = w.ch0;
        auto fetch = [&](int kind, int c0) {
          __syncwarp();
          const char* pool = kind ? a.kv.v + ch0 * 4 : a.kv.k;
          const int width = kind ? widths[1] : widths[0];
#pragma unroll
          for (int i = 0; i < GROUPS; ++i) {
            const long long o = __shfl_sync(0xffffffffu, off, i * 4 + lane / 8);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int c = c0 + h * 8 + (lane & 7);
              x[h][i][0] = x[h][i][1] = make_float4(0.f, 0.f, 0.f, 0.f);
              if (o >= 0 && c * 8 < width) {
                x[h][i][0] = load4((const float*)(pool + o) + c * 8);
                x[h][i][1] = load4((const float*)(pool + o) + c * 8 + 4);
              }
            }
          }
        };
        fetch(0, 0);
#pragma unroll 1
        for (int t = w.lo; t < hi && ok; ++t, ++it, k_ring.next(), v_ring.next()) {
#pragma unroll 1
          for (int kind = 0; kind < 2; ++kind) {  // keys, values
            const int slot = kind ? v_ring.at : k_ring.at, n = ((kind ? widths[1] : widths[0]) + 15) / 16 * 2;
            if (kind ? it >= VS && !(ok = wait(s.vempty[slot], v_ring.turn ^ 1))
                     : it >= KS && !(ok = wait(s.kempty[slot], k_ring.turn ^ 1)))
              break;
            const uint32_t to = kind ? v0 + slot * S::kVSlot : k0 + slot * S::kKSlot;
            const bool look = kind && (t + 1) * TK > len;
            uint32_t marks[TK / 32] = {};
#pragma unroll 1
            for (int c0 = 0; c0 < n; c0 += 16) {  // the same for all lanes: they exchange the rows' places
#pragma unroll
              for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < GROUPS; ++i) {
                  const int r = row_of(i) + lane / 8, c = c0 + h * 8 + (lane & 7);
                  if (r >= TK || c >= n) continue;
                  float y[8] = {x[h][i][0].x, x[h][i][0].y, x[h][i][0].z, x[h][i][0].w,
                                x[h][i][1].x, x[h][i][1].y, x[h][i][1].z, x[h][i][1].w};
                  if (look && t * TK + r >= len) {
                    bool bad = false;
#pragma unroll
                    for (int j = 0; j < 8; ++j) bad |= !(fabsf(y[j]) < INFINITY);
                    if (bad) {
#pragma unroll
                      for (int j = 0; j < 8; ++j) y[j] = 0.f;
#pragma unroll
                      for (int j = 0; j < TK / 32; ++j)
                        if (r >> 5 == j) marks[j] |= 1u << (r & 31);
                    }
                  }
                  uint4 parts[3];
                  cut8(y, parts);
                  const uint32_t dst = to + swizzled(c, r, TK);
#pragma unroll
                  for (int j = 0; j < 3; ++j) sts16(dst + j * (kind ? S::kVPart : S::kKPart), parts[j]);
                }
              // the next step's are on their way while this one is waited for
              if (c0 + 16 < n) {
                fetch(kind, c0 + 16);
              } else if (kind == 0) {
                fetch(1, 0);
              } else if (t + 1 < hi) {
                off = place_of(t + 1, page);
                page = page_of(t + 2);
                fetch(0, 0);
              }
            }
            __syncwarp();
            if (look) {
#pragma unroll
              for (int i = 0; i < TK / 32; ++i) {
                marks[i] = __reduce_or_sync(0xffffffffu, marks[i]);
                if (lane == 0) s.vbad[slot][loader][i] = marks[i];
              }
            }
            signal(kind ? s.vfull[slot] : s.kfull[slot]);
            if (look) arrive(s.looked[slot]);
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (s.waits.abort && threadIdx.x == 0) {  // no warp can give up from here on
    // nor is a copy under way when the CTA's memory goes: they take microseconds
    const unsigned long long t0 = globaltimer();
    while (globaltimer() - t0 < 2000000ull) {
    }
    a.cut[blockIdx.x].live = -1;
    kv_report(a.status, ER_KV_GAVE_UP);
  }
  if (warp == kIssueWarp) tmem_dealloc<1>(tmem, 512);
}

template <typename S, typename TC, typename TQ>
int tree_launch(const TreeArgs& a, const CUtensorMap* maps, cudaStream_t st) {
  static std::atomic<unsigned long long> allowed;
  const int smem = S::kSmem + 1024;
  if (int rc = allow_smem(kv_tree_kernel<S, TC, TQ>, smem, allowed)) return rc;
  return kv_launch(kv_tree_kernel<S, TC, TQ>, dim3(a.grid), S::kThreads, smem, false, st, "kv_tree_kernel", a, maps[0],
                   maps[1]);
}

}  // namespace
}  // namespace er
