// Decode attention of one layer for sequences that share a prefix (etxb_attn_shared): a group of sequences has one block table for the positions
// they have in common and each sequence one for its own.
//
//   out_b,h = sum_i p_i v_i / sum_i p_i,  p_i = exp(scale * q_b,h . k_i - m),  i over the prefix of b's group and b's own positions
//
// Work.  A unit is a set of up to 128 rows (q heads of sequences) and the positions they attend to: the rows of up to 128 / G sequences of a group and one
// kv head over the group's prefix, or the G rows of one sequence and kv head over its own positions.  A unit's positions go in tiles of TP (128; 64 above
// 128 elements per head).  All tiles of the call in one order are shared out evenly: CTA w takes [w T / W, (w + 1) T / W), so that one long prefix fills the
// device and short contexts do not leave it idle.  Where a share ends inside a unit, both parts (segments) leave fp32 partial results -- sum of p v, sum of p,
// m -- which a second kernel joins; the prefix's and a sequence's own parts meet there as well.
//
// A tile on the tensor cores (tcgen05, fp32 accumulators in tensor memory):
//   S = Q K^T   M = 128 rows, operands in shared memory without swizzle.  A page of keys, [HD / 8][16 positions][8], IS a column of core matrices, 8 positions x
//               16 bytes each, so whole pages are bulk copies and are multiplied as they lie: one instruction takes positions 0 .. 7 of every page of the tile
//               (the stride between 8-row groups is a page), another positions 8 .. 15.
//   softmax     a thread has a row: it reads its scores from tensor memory, keeps the running maximum and sum, and writes P over S.
//   O += P V    A from tensor memory; a page of values, [HD][16 positions], is 32-byte rows with the positions inside: a TMA tensor copy with SWIZZLE_32B makes it
//               the K-major operand of one k16 step.
// P goes in as two bf16 numbers, P = hi + lo, both cut off: 16 bits.  One would round every probability by 2^-9, which contexts
// of few positions show in the output; the second product is 512 clocks of tensor pipe a tile, beside the 2900 clocks that a tile's bytes take from HBM.
//
// Roles: two sets of eight warps of softmax, which have alternate tiles, half a row a thread; a warp that copies keys and values into a ring of tiles; a thread that
// issues Q K^T; a warp that waits for the values, clears those behind the last position (whatever the cache holds there, 0 times it must be 0) and issues P V; a warp
// that works out the worker's segments and fetches the rows of their Q.  They meet at mbarriers only, and three tiles of scores, each with its P in place, are on their way
// at once, so products, softmax and copies of neighbouring tiles and segments overlap.  Every wait is bounded, and every role waits for every phase of a barrier.
//
// Measured (32 q heads of 128): 2 sequences over 131000 shared positions, 8 kv heads, 125 us, 4.3 TB/s (539 MB: 83 us); 64 over 32500 103 us (199 MB: 30 us; products: 21);
// 32 over 8150, 4 kv heads, 35 us; 4 over 1024 19 us, mostly the host's.  Of 256 elements, 4 kv heads: 16 sequences over 32500 67 us (148 MB: 23 us), in tiles of 64 positions.  A tile takes 2900 to 3000 clocks: its bytes 2900 from HBM with all SMs at it, its products 1800.  Tried and slower: one set of softmax warps; P in columns of its own (softmax waits for P V);
// the second kernel launched ahead of the first one's end (its blocks wait on the SMs).  Contexts of their own, a short segment each, take 4500 clocks a tile, most of it the way from Q to the first product.
#include <cuda.h>
#include <cuda_bf16.h>
#include <stdio.h>
#include <string.h>

#include "etxb_host.h"

namespace etxb_shared {

constexpr int BS = 16, ROWS = 128, OWN_ROWS = 16, MAX_SLOTS = 16;
constexpr int SETS = 2, SET_WARPS = 8, W_COPY = 16, W_QK = 17, W_PV = 18, W_Q = 19, THREADS = 640;
constexpr unsigned long long WAIT_NS = 2000000000ull;

struct Groups { int32_t first[ETXB_SHARED_MAX_SEQS + 1]; };

// What both kernels derive alike from the sizes: where a unit's partial results lie.
struct Layout {
  int G, spt;                 // q heads per kv head; sequences whose rows fill a unit of a prefix
  int tp;                     // positions of a tile
  int workers;
  int prows;                  // rows of the largest unit of a prefix
  int slots, qrows;           // of the kernel's shared memory: tiles of keys or values in the ring (even), rows of Q kept for a prefix
  int punits;                 // units of prefixes, counted generously (see prefix_unit); a unit's parts have the numbers unit + worker
  long long pslots, oslots;   // numbers of parts of prefixes / of own positions
  float* pO; float* pml; float* oO; float* oml;      // of a part [HD / 4][rows][4], [rows][2] (m in units of log2, l), from the row on that part_row names
  int32_t* hdr;               // [pslots + oslots]: status bits of a segment
  int32_t* gave_up;           // [workers]: not 0 where one did
  int32_t* of;                // [units][2]: first and last worker that has tiles of a unit
};

struct Params {
  etxb_attn_shared_args a;
  Layout y;
  Groups groups;
  CUtensorMap vmap;
};

// ------------------------------------------------------------------------------------------------ primitives
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint64_t* b, uint32_t n) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(b)), "r"(n) : "memory"); }
__device__ __forceinline__ void bar_arrive(uint64_t* b) { asm volatile("{\n\t.reg .b64 s;\n\tmbarrier.arrive.shared::cta.b64 s, [%0];\n\t}" ::"r"(smem_u32(b)) : "memory"); }
__device__ __forceinline__ void bar_expect(uint64_t* b, uint32_t bytes) {
  asm volatile("{\n\t.reg .b64 s;\n\tmbarrier.arrive.expect_tx.shared::cta.b64 s, [%0], %1;\n\t}" ::"r"(smem_u32(b)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint64_t* b, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(smem_u32(b)), "r"(parity) : "memory");
  return ok != 0;
}
__device__ __forceinline__ unsigned long long now_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
// Waits for phase `n` (0, 1, ..) of a barrier; false, for everyone from then on, when it takes two seconds.  (The clock is looked at once in 256 tries:
// reading it takes longer than most waits.  The loop is not inlined: some twenty waits, and the roles together have to fit the code that an SM keeps.)
__device__ __noinline__ bool bar_wait_on(uint32_t bar, uint32_t parity, volatile int* stop) {
  unsigned long long t0 = 0;
  for (uint32_t i = 1;; ++i) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    if (ok) return true;
    if ((i & 255) == 0) {
      const unsigned long long t = now_ns();
      if (t0 == 0) t0 = t;
      if (*stop) return false;
      if (t - t0 > WAIT_NS) { *stop = 1; return false; }
    }
  }
}
__device__ __forceinline__ bool bar_wait(uint64_t* b, uint32_t n, volatile int* stop) { return bar_try(b, n & 1) || bar_wait_on(smem_u32(b), n & 1, stop); }
// Waits for a phase whatever the others do, for what a block has on its way before it ends (with the same limit).
__device__ __noinline__ void bar_drain(uint32_t bar, uint32_t parity) {
  const unsigned long long t0 = now_ns();
  uint32_t ok = 0;
  while (!ok) {
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    if (now_ns() - t0 > WAIT_NS) break;
  }
}
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int y, int z, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
               ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(0), "r"(y), "r"(z) : "memory");
}
// Shared-memory matrix descriptor, K-major.  swizzle 0: core matrices of 8 rows x 16 bytes, lbo between those that follow in k, sbo between groups of 8 rows;
// 6: rows of 32 bytes swizzled in pairs of 16, groups of 8 rows sbo apart.
__device__ __forceinline__ uint64_t desc(uint32_t addr, uint32_t lbo, uint32_t sbo, uint32_t swizzle) {
  return (uint64_t)((addr & 0x3ffffu) >> 4) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(sbo >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)swizzle << 61);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accum) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accum) : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
#define ETXB_R8(r, o) "=r"(r[o]), "=r"(r[o + 1]), "=r"(r[o + 2]), "=r"(r[o + 3]), "=r"(r[o + 4]), "=r"(r[o + 5]), "=r"(r[o + 6]), "=r"(r[o + 7])
#define ETXB_W8(r, o) "r"(r[o]), "r"(r[o + 1]), "r"(r[o + 2]), "r"(r[o + 3]), "r"(r[o + 4]), "r"(r[o + 5]), "r"(r[o + 6]), "r"(r[o + 7])
// 32 / 16 columns of this warp's lanes; the loads are asynchronous until tmem_wait_ld
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, "
               "%27, %28, %29, %30, %31}, [%32];" : ETXB_R8(r, 0), ETXB_R8(r, 8), ETXB_R8(r, 16), ETXB_R8(r, 24) : "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               : ETXB_R8(r, 0), ETXB_R8(r, 8) : "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
               ::"r"(addr), ETXB_W8(r, 0), ETXB_W8(r, 8) : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ bool elect() {
  uint32_t e;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
  return e != 0;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ uint64_t pack2(uint32_t lo, uint32_t hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(hi));
  return d;
}
__device__ __forceinline__ uint64_t pack2(float lo, float hi) { return pack2(__float_as_uint(lo), __float_as_uint(hi)); }
__device__ __forceinline__ void unpack2(uint64_t v, float& lo, float& hi) {
  uint32_t a, b;
  asm("mov.b64 {%0, %1}, %2;" : "=r"(a), "=r"(b) : "l"(v));
  lo = __uint_as_float(a); hi = __uint_as_float(b);
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// ------------------------------------------------------------------------------------------------ shares
// Tiles before group g / sequence b in the order of all tiles: the prefixes' units (group, kv head, rows), then the sequences' (sequence, kv head).
struct Cum {
  int32_t* p;                 // [groups + 1]
  int32_t* s;                 // [seqs + 1]
  int32_t* len;               // [groups], [seqs]
};
__device__ __forceinline__ bool bad_length(int len, int width) { return len < 0 || len > width * BS; }
__device__ __forceinline__ int tiles_of(int len, int width, int tp) { return bad_length(len, width) ? 0 : (len + tp - 1) / tp; }
__device__ __forceinline__ int units_of(const Params& P, int g) { return (P.groups.first[g + 1] - P.groups.first[g] + P.y.spt - 1) / P.y.spt; }

// Fills c (warps 0 and 1; the caller's barrier follows).
__device__ __forceinline__ void cumulate(const Params& P, const Cum& c) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (warp > 1) return;
  const etxb_attn_shared_args& a = P.a;
  const int n = warp == 0 ? a.groups : a.seqs, width = warp == 0 ? a.prefix_width : a.table_width;
  const int32_t* lens = warp == 0 ? a.prefix_lens : a.lens;
  int32_t* out = warp == 0 ? c.p : c.s;
  int32_t* len = warp == 0 ? c.len : c.len + a.groups;
  int base = 0;
  for (int i0 = 0; i0 < n; i0 += 32) {
    const int i = i0 + lane;
    int v = 0;
    if (i < n) {
      len[i] = lens[i];
      v = tiles_of(len[i], width, P.y.tp) * a.NKV;
      if (warp == 0) v *= units_of(P, i);
    }
    int s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int x = __shfl_up_sync(~0u, s, o); if (lane >= o) s += x; }
    if (i < n) out[i] = base + s - v;
    base += __shfl_sync(~0u, s, 31);
  }
  if (lane == 0) out[n] = base;
}
__device__ __forceinline__ int find(const int32_t* c, int n, int t) {      // the last i with c[i] <= t whose successor is above t
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (c[mid] <= t) lo = mid; else hi = mid - 1;
  }
  return lo;
}
// The first tile of worker w: floor(total * w / workers), without 64-bit arithmetic (workers <= 256).
__device__ __forceinline__ int share(int total, int w, int workers) {
  const int q = total / workers, r = total - q * workers;
  return q * w + r * w / workers;
}

// Tiles [t0, t1) of a worker.  Tiles of prefixes and of sequences' own positions have workers of their own, as many as their time asks for: a tile of own
// positions, in short units, takes OWN_COST / PREFIX_COST times as long as one of a prefix (64 sequences over 32500 positions, 500 of their own, 8 kv heads of 128, in a graph: 2 : 3 98 us, 1 : 1 113, 1 : 2 104;
// other shapes take the same, which was not measured for them).  No worker among those that share is without a tile.
constexpr int PREFIX_COST = 2, OWN_COST = 3;
__device__ __forceinline__ void share_of(int tp, int to, int W, int w, int& t0, int& t1) {
  int wp = tp, wo = to;                                             // fewer tiles than workers: one each
  if ((unsigned)tp + (unsigned)to > (unsigned)W) {
    const float cp = (float)tp * PREFIX_COST, co = (float)to * OWN_COST;
    wp = min(tp, max(tp > 0 ? 1 : 0, min(to > 0 ? W - 1 : W, (int)((float)W * cp / (cp + co) + 0.5f))));
    wo = min(to, W - wp);
    wp = min(tp, W - wo);                                           // (what the sequences do not need)
  }
  t0 = t1 = 0;
  if (w < wp) { t0 = share(tp, w, wp); t1 = share(tp, w + 1, wp); }
  else if (w < wp + wo) { t0 = tp + share(to, w - wp, wo); t1 = tp + share(to, w - wp + 1, wo); }
}

// The first row of worker w's part of a unit whose rows have row0 others of units before them: parts of one unit lie `most` rows apart, the largest unit's number, and a
// worker's part of the next unit begins at least the unit's own rows behind its part of this one.  (With `most` rows for every part, one large group beside a
// thousand of one sequence took 567 MB for 43.)
__device__ __forceinline__ long long part_row(int row0, int most, int w) { return (long long)row0 + (long long)most * w; }

// The first unit of group g's prefix: no more units lie before it than sequences / spt + groups, for each kv head.
__device__ __forceinline__ int prefix_unit(const Params& P, int g) { return (P.groups.first[g] / P.y.spt + g) * P.a.NKV; }

struct Segment {
  int n;                      // tiles of the unit from tile0 on
  int own;                    // a sequence's own positions, not a prefix's
  int h;                      // kv head
  int seq0, rows;             // first sequence and number of rows
  int tile0, ends;            // the unit's last tile is in it
  int len;                    // positions of the unit
  int unit;                   // of all units, prefixes' first; its parts have the numbers unit + worker
  int row0;                   // rows of the units before it, prefixes' or own positions'
  const int32_t* table;
};
__device__ __forceinline__ void segment_at(const Params& P, const Cum& c, int t, int end, Segment& s) {
  const etxb_attn_shared_args& a = P.a;
  const int tp_all = c.p[a.groups];
  int per;
  s.own = t >= tp_all;
  if (!s.own) {
    const int g = find(c.p, a.groups, t), mt = units_of(P, g), first = P.groups.first[g];
    per = (c.p[g + 1] - c.p[g]) / (mt * a.NKV);
    const int rel = t - c.p[g], unit = rel / per;
    s.h = unit / mt;
    const int m = unit - s.h * mt;
    s.seq0 = first + m * P.y.spt;
    s.rows = min(P.y.spt, P.groups.first[g + 1] - s.seq0) * P.y.G;
    s.tile0 = rel - unit * per;
    s.len = c.len[g];
    s.table = a.prefix_tables + g * a.prefix_stride;
    s.unit = prefix_unit(P, g) + unit;
    s.row0 = (first * a.NKV + s.h * (P.groups.first[g + 1] - first) + m * P.y.spt) * P.y.G;
  } else {
    const int r = t - tp_all, b = find(c.s, a.seqs, r);
    per = (c.s[b + 1] - c.s[b]) / a.NKV;
    const int rel = r - c.s[b];
    s.h = rel / per;
    s.seq0 = b; s.rows = P.y.G;
    s.tile0 = rel - s.h * per;
    s.len = c.len[a.groups + b];
    s.table = a.tables + b * a.table_stride;
    s.unit = P.y.punits + b * a.NKV + s.h;
    s.row0 = (b * a.NKV + s.h) * P.y.G;
  }
  s.n = min(per - s.tile0, end - t);
  s.ends = s.tile0 + s.n == per;
}

// ------------------------------------------------------------------------------------------------ the tiles
constexpr int SEGS = 8;                       // segments known ahead
struct Shared {
  uint64_t full[MAX_SLOTS], empty[MAX_SLOTS];       // ring of key / value tiles: K0 K1 V0 K2 V1 .. (V of tile n: use 2 n + 2)
  uint64_t s_full[3], p_full[3], pv_done[3], o_full[SETS], o_free, q_full[4], q_free[4], seg_full[SEGS], seg_free[SEGS], pair[SETS][4], m_full[3][4], drained[2];
  Segment seg[SEGS];
  float part[SETS][2][2][ROWS];               // maxima that the two warps of a row tell each other: by set, turn, half
  float m[3][ROWS];                           // each row's maximum after tile n, at n % 3
  float2 l[2][SETS][2][ROWS];                 // a set's sums of a segment and the maximum they are relative to: by turn of segments, set, half
  uint32_t tmem;
  int stop;
};

// Dynamic shared memory: the ring (y.slots tiles), Q (y.qrows rows, four sequences' at least), the tiles before each group and sequence and their lengths.
// The number of slots is even: values always lie in the even slots, so that whoever looks at values alone sees every use of its slots (but the first of slot
// 0).  Behind it all 2 KB: an instruction reads 128 rows of Q, and where there are fewer the last ones lie behind the buffer.
__host__ __device__ __forceinline__ int q_size(int hd, int qrows) { return (qrows > 4 * OWN_ROWS ? qrows : 4 * OWN_ROWS) * hd * 2; }
template <int TP>
__global__ void __launch_bounds__(THREADS, 1) tiles_kernel(const __grid_constant__ Params P) {
  extern __shared__ __align__(256) unsigned char dyn[];
  __shared__ Shared sh;
  constexpr int PAGES = TP / BS, HALF = TP / 2;                     // pages of a tile; columns of S that one half of the pages' positions take
  constexpr int C_O = 3 * TP;                                       // columns of tensor memory: three tiles of S, over which P is written, then O
  const etxb_attn_shared_args& a = P.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, HD = a.HD, worker = blockIdx.x;
  const uint32_t page_bytes = (uint32_t)HD * BS * 2, q_bytes = q_size(HD, P.y.qrows), slot_bytes = PAGES * page_bytes, SLOTS = P.y.slots;
  unsigned char* const base = (unsigned char*)(((uintptr_t)dyn + 255) & ~(uintptr_t)255);
  unsigned char* const qbuf = base + SLOTS * slot_bytes;
  const Cum cum = {(int32_t*)(qbuf + q_bytes), (int32_t*)(qbuf + q_bytes) + a.groups + 1, (int32_t*)(qbuf + q_bytes) + a.groups + a.seqs + 2};
  volatile int* const stop = &sh.stop;

  cumulate(P, cum);
  if (tid == W_Q * 32) {
    for (int i = 0; i < SLOTS; ++i) { bar_init(&sh.full[i], 1); bar_init(&sh.empty[i], 1); }
    for (int i = 0; i < 3; ++i) { bar_init(&sh.s_full[i], 1); bar_init(&sh.p_full[i], SET_WARPS); bar_init(&sh.pv_done[i], 1); }
    for (int i = 0; i < 12; ++i) bar_init(&sh.m_full[i / 4][i % 4], 1);
    for (int i = 0; i < SETS; ++i) { bar_init(&sh.o_full[i], 1); bar_init(&sh.drained[i], 1); }
    bar_init(&sh.o_free, SET_WARPS);
    for (int i = 0; i < 4; ++i) { bar_init(&sh.q_full[i], 32); bar_init(&sh.q_free[i], 1); bar_init(&sh.pair[0][i], 2); bar_init(&sh.pair[1][i], 2); }
    for (int i = 0; i < SEGS; ++i) { bar_init(&sh.seg_full[i], 1); bar_init(&sh.seg_free[i], SETS * SET_WARPS + 3); }
    sh.stop = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == W_QK) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sh.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    fence_before();
  }
  fence_async();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sh.tmem;
  int t0, t1;
  share_of(cum.p[a.groups], cum.s[a.seqs], P.y.workers, worker, t0, t1);
  // A role's next segment (false: a wait ran out), and the end of its use.
  auto next_segment = [&](uint32_t k, Segment& s) {
    if (!bar_wait(&sh.seg_full[k % SEGS], k / SEGS, stop)) return false;
    s = sh.seg[k % SEGS];
    return true;
  };

  if (warp < SETS * SET_WARPS) {
    // ---- softmax: set n % 2 has tile n, so that one set's waits are the other's work.  In a set, a row belongs to a lane of two warps, each of which has half
    // of the tile's positions: blocks of 16 columns of S in both halves.
    constexpr int MINE = TP / 2;                                    // positions of a warp
    const int set = warp / SET_WARPS, quarter = warp & 3, hf = (warp >> 2) & 1, row = quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    // scores in units of log2 (a scale of 0 as the least there is: a masked score stays minus infinity)
    const float sl = fmaxf(a.scale * 1.4426950408889634f, 1e-37f);
    uint32_t n = 0, seg = 0, turn = 0, outs = 0;                    // tiles and segments so far, of both sets; exchanges, and segments that this set wrote out
    float m = -INFINITY, l = 0.f;                                   // the row's maximum, and this warp's sum relative to it
    bool ok = true;
    for (int t = t0; t < t1 && ok; ++seg) {
      Segment s;
      ok = __all_sync(~0u, next_segment(seg, s));
      const bool busy = quarter * 32 < s.rows;                      // (a warp without rows only keeps the others' time)
      const int mine = set ^ (n & 1);                               // the first tile of this segment that is the set's
      m = -INFINITY; l = 0.f;
      for (int i = mine; i < s.n && ok; i += 2) {
        const uint32_t tile = n + i, sb = tile % 3, scol = tmem + lanes + sb * TP + hf * (MINE / 2);
        ok = bar_wait(&sh.s_full[sb], tile / 3, stop);
        ok = __all_sync(~0u, ok);
        if (!ok) break;
        fence_after();
        if (busy) {
          const int valid = s.len - (s.tile0 + i) * TP - hf * MINE;
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
          for (int j = 0; j < MINE / 32; ++j) {                     // 32 positions: page 2 j + k / 8, half h of it, its position k % 8 (k < 16)
            uint32_t r[32];
            tmem_ld16(scol + 16 * j, r);
            tmem_ld16(scol + HALF + 16 * j, r + 16);
            tmem_wait_ld();
            const int left = valid - 32 * j;
            if (left < 32) {                                        // scores behind the last position become minus infinity
#pragma unroll
              for (int c = 0; c < 32; ++c) if (c % 16 / 8 * 16 + c / 16 * 8 + c % 8 >= left) r[c] = 0xff800000u;
              tmem_st16(scol + 16 * j, r);
              tmem_st16(scol + HALF + 16 * j, r + 16);
              tmem_wait_st();
            }
#pragma unroll
            for (int c = 0; c < 32; c += 8)
#pragma unroll
              for (int k = 0; k < 4; ++k) mx[k] = fmaxf(mx[k], fmaxf(__uint_as_float(r[c + 2 * k]), __uint_as_float(r[c + 2 * k + 1])));
          }
          float mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
          // the other warp's, and the maximum after the tile before
          sh.part[set][turn & 1][hf][row] = mt;
          __syncwarp();
          if (lane == 0) bar_arrive(&sh.pair[set][quarter]);
          ok = bar_wait(&sh.pair[set][quarter], turn, stop);
          if (tile > 0) ok = ok && bar_wait(&sh.m_full[(tile - 1) % 3][quarter], (tile - 1) / 3, stop);
          ok = __all_sync(~0u, ok);
          if (!ok) break;
          mt = fmaxf(mt, sh.part[set][turn & 1][hf ^ 1][row]);
          ++turn;
          const float m0 = i == 0 ? -INFINITY : sh.m[(tile - 1) % 3][row];
          // the maximum moves only when the new one is above it by a factor of 2^8 or more: till then probabilities of up to 2^8 do no harm
          const bool up = row < s.rows && m0 != -INFINITY && (mt - m0) * sl > 8.f;
          const float m1 = up || m0 == -INFINITY ? mt : m0;
          if (hf == 0) {
            sh.m[sb][row] = m1;
            __syncwarp();
            if (lane == 0) bar_arrive(&sh.m_full[sb][quarter]);
          }
          if (m1 != m) { l = l == 0.f ? 0.f : l * ex2((m - m1) * sl); m = m1; }
          if (__any_sync(~0u, up)) {
            const float f = up ? ex2((m0 - m1) * sl) : 1.f;
            ok = bar_wait(&sh.pv_done[(tile - 1) % 3], (tile - 1) / 3, stop);
            ok = __all_sync(~0u, ok);
            if (!ok) break;
            fence_after();
            const uint32_t ocol = tmem + lanes + C_O;
            const int mid = (HD / 16 + 1) / 2 * 16;
#pragma unroll 1
            for (int c = hf ? mid : 0; c < (hf ? HD : mid); c += 16) {
              uint32_t o[16];
              tmem_ld16(ocol + c, o);
              tmem_wait_ld();
#pragma unroll
              for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
              tmem_st16(ocol + c, o);
            }
          }
          const float ms = m == -INFINITY ? 0.f : m * sl;
          const uint64_t sl2 = pack2(sl, sl), ms2 = pack2(-ms, -ms), c2 = pack2(1.0f + 0x1p-17f, 1.0f + 0x1p-17f);
          uint64_t ls[2] = {0, 0};
          // two pages at a time, over whose scores 16 columns of hi and 16 of lo are written (pages behind the last are not multiplied).  The scores are read
          // twice, and in loops: more registers would cost warps, and code that an SM does not keep costs more.
#pragma unroll 1
          for (int j = 0; j < MINE / 32 && 32 * j < valid; ++j) {
            uint32_t a0[16], a1[16];
            tmem_ld16(scol + 16 * j, a0);
            tmem_ld16(scol + HALF + 16 * j, a1);
            tmem_wait_ld();
            uint32_t hi[16], lo[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {                          // positions 2 k and 2 k + 1
              const int pos = 2 * k, c = pos / 16 * 8 + pos % 8;
              const uint64_t v = (pos & 8) ? pack2(a1[c], a1[c + 1]) : pack2(a0[c], a0[c + 1]);
              float p0, p1, y0, y1;
              unpack2(fma2(v, sl2, ms2), p0, p1);
              p0 = ex2(p0); p1 = ex2(p1);
              const uint64_t p = pack2(p0, p1);
              ls[k & 1] = add2(ls[k & 1], p);
              // hi: the upper 16 bits; lo: the upper 16 bits of what is left and 2^-17 of p more -- what the cut takes off on the average, and so that lo
              // is never 0 where p is not (0 x inf would spoil the sum of an infinite value) nor negative
              const uint32_t u0 = __float_as_uint(p0), u1 = __float_as_uint(p1);
              unpack2(fma2(p, c2, pack2((u0 & 0xffff0000u) ^ 0x80000000u, (u1 & 0xffff0000u) ^ 0x80000000u)), y0, y1);
              hi[k] = __byte_perm(u0, u1, 0x7632);
              lo[k] = __byte_perm(__float_as_uint(y0), __float_as_uint(y1), 0x7632);
            }
            tmem_st16(scol + 16 * j, hi);
            tmem_st16(scol + HALF + 16 * j, lo);
          }
          {
            float x, y;
            unpack2(add2(ls[0], ls[1]), x, y);
            l += x + y;
          }
          if (i + 2 >= s.n) sh.l[seg & 1][set][hf][row] = make_float2(m, l);
          tmem_wait_st();
        } else if (hf == 0 && lane == 0) bar_arrive(&sh.m_full[sb][quarter]);
        fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(&sh.p_full[sb]);
        if (i + 1 < s.n) continue;
        // the unit's part in this segment: its set of the last tile writes it out, when the other set's warps have left their sums
        if (busy) {
          if (lane == 0) bar_arrive(&sh.pair[set][quarter]);
          ok = bar_wait(&sh.pair[set][quarter], turn++, stop);
        }
        ok = ok && bar_wait(&sh.o_full[set], outs++, stop);
        if (s.n > 1) ok = ok && bar_wait(&sh.p_full[(tile - 1) % 3], (tile - 1) / 3, stop);
        ok = __all_sync(~0u, ok);
        fence_after();
        const int mid = (HD / 16 + 1) / 2 * 16, c0 = hf ? mid : 0, c1 = hf ? HD : mid;           // this warp's columns
        const int stride = s.rows;
        const long long at = part_row(s.row0, s.own ? P.y.G : P.y.prows, worker);
        const bool writes = ok && row < s.rows;
        float* O = (s.own ? P.y.oO : P.y.pO) + at * HD + (size_t)row * 4;
#pragma unroll 1
        for (int c = c0; c < c1; c += 32) {
          uint32_t r[32];
          if (ok && busy) {
            tmem_ld16(tmem + lanes + C_O + c, r);
            if (c + 16 < c1) tmem_ld16(tmem + lanes + C_O + c + 16, r + 16);
            tmem_wait_ld();
          }
          if (writes) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
              if (c + 4 * k < c1) *(uint4*)(O + (size_t)(c / 4 + k) * stride * 4) = make_uint4(r[4 * k], r[4 * k + 1], r[4 * k + 2], r[4 * k + 3]);
          }
        }
        fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(&sh.o_free);
        if (writes && hf == 0) {
          float L = 0.f;
#pragma unroll
          for (int x = 0; x < 4; ++x) {                             // the set's own two, then the other's
            if (x >= 2 && s.n == 1) break;
            const float2 p = sh.l[seg & 1][set ^ (x >> 1)][x & 1][row];
            if (p.y != 0.f) L += p.x == m ? p.y : p.y * ex2((p.x - m) * sl);
          }
          *((float2*)(s.own ? P.y.oml : P.y.pml) + at + row) = make_float2(m == -INFINITY ? m : m * sl, L);
        }
      }
      n += s.n;
      __syncwarp();
      if (lane == 0) bar_arrive(&sh.seg_free[seg % SEGS]);
      t += s.n;
    }
  } else if (warp == W_COPY) {
    // ---- copies: a lane per page
    uint32_t use = 0, sl = 0, round = 0, seg = 0, left_out = ~0u;    // running number of ring slots taken, the next one, how often it was before; a use without a copy
    bool ok = true, have = false;
    int vp = 0, vn = 0, vh = 0;                                     // the tile whose values follow
    auto put = [&](int n_pages, int page, int h, bool values) {
      if (round > 0) ok = ok && bar_wait(&sh.empty[sl], round - 1, stop);
      ok = __all_sync(~0u, ok);
      if (!ok) return;
      if (lane == 0) bar_expect(&sh.full[sl], n_pages * page_bytes);
      __syncwarp();
      unsigned char* dst = base + sl * slot_bytes + lane * page_bytes;
      if (lane < n_pages) {
        if (values) tma_load_3d(dst, &P.vmap, h * HD, page, &sh.full[sl]);
        else bulk_load(dst, (const __nv_bfloat16*)a.kc + page * a.k_stride + (long long)h * HD * BS, page_bytes, &sh.full[sl]);
      }
      ++use;
      if (++sl == SLOTS) { sl = 0; ++round; }
    };
    for (int t = t0; t < t1 && ok; ++seg) {
      Segment s;
      ok = __all_sync(~0u, next_segment(seg, s));
      if (!ok) break;
      const int first = s.tile0 * PAGES, pages = min(s.n * PAGES, (s.len + BS - 1) / BS - first);
      int bad = 0;
      // the numbers of 32 pages at a time, the next ones on their way
      int ids = lane < pages ? s.table[first + lane] : 0, more = 0;
      for (int p0 = 0; p0 < pages && ok; p0 += PAGES) {
        if (p0 % 32 == 0) {
          if (p0 > 0) ids = more;
          if (p0 + 32 + lane < pages) more = s.table[first + p0 + 32 + lane];
          const bool off = p0 + lane < pages && (ids < 0 || ids >= a.pages);
          if (off) ids = 0;
          if (__any_sync(~0u, off)) bad = ETXB_SHARED_BAD_PAGE;
        }
        const int np = min(PAGES, pages - p0), page = __shfl_sync(~0u, ids, (p0 + lane) & 31);
        put(np, page, s.h, false);
        if (have) put(vn, vp, vh, true);
        have = true; vp = page; vn = np; vh = s.h;
      }
      if (lane == 0) {
        P.y.hdr[(s.own ? P.y.pslots - P.y.punits : 0) + s.unit + worker] = bad;
        if (s.tile0 == 0) P.y.of[2 * s.unit] = worker;
        if (s.ends) P.y.of[2 * s.unit + 1] = worker;
        if (bad && a.status) atomicOr(a.status, bad);
        bar_arrive(&sh.seg_free[seg % SEGS]);
      }
      t += s.n;
    }
    if (have && ok) {                                               // the use behind the last K is left out
      left_out = use++;
      if (++sl == SLOTS) { sl = 0; ++round; }
      put(vn, vp, vh, true);
    }
    // before the block ends, nothing is on its way into its memory any more (also when it gave up, before or behind the use without a copy): the last copy
    // into every slot.  (Earlier ones have come: a slot is taken again when it was read.)
    for (uint32_t u = use > SLOTS + 2 ? use - SLOTS - 2 : 0; u < use; ++u) {
      if (u == left_out || (u + SLOTS < use && u + SLOTS != left_out)) continue;
      bar_drain(smem_u32(&sh.full[u % SLOTS]), (u / SLOTS) & 1);
    }
  } else if (warp == W_QK) {
    // ---- S = Q K^T: one thread, and another one for O += P V, so that neither waits behind what the other waits for
    if (elect()) {
      const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(ROWS >> 4) << 24);
      uint32_t n = 0, seg = 0, sl = 0, round = 0;                     // (K of tile n is use 2 n - 1, but 0 for the first)
      bool ok = true;
      for (int t = t0; t < t1 && ok; ++seg) {
        Segment s;
        ok = next_segment(seg, s);
        ok = ok && bar_wait(&sh.q_full[seg & 3], seg >> 2, stop);
        // (a sequence's own rows lie close together: what the other rows of the instruction read there reaches accumulator rows that nobody reads)
        const uint32_t qrows = s.own ? OWN_ROWS : P.y.qrows;
        const uint64_t ad = desc(smem_u32(qbuf + (s.own ? (seg & 3) * (OWN_ROWS * (uint32_t)HD * 2) : 0u)), qrows * 16, 128, 0), astep = 2 * qrows;
        for (int i = 0; i < s.n && ok; ++i, ++n) {
          const int np = min(PAGES, (s.len + BS - 1) / BS - (s.tile0 + i) * PAGES);
          const uint32_t sb = n % 3;
          if (n >= 3) ok = bar_wait(&sh.pv_done[sb], n / 3 - 1, stop);               // (P of tile n - 3 lies where S of this one goes)
          ok = ok && bar_wait(&sh.full[sl], round, stop);
          if (!ok) break;
          fence_after();
          const uint32_t id = idesc | ((uint32_t)((np + 1) & ~1) << 17);             // N = 8 positions of each page, a multiple of 16
          const uint32_t d = tmem + sb * TP;
          const uint64_t b0 = desc(smem_u32(base + sl * slot_bytes), 256, page_bytes, 0);
#pragma unroll 1
          for (int k = 0; k < HD / 16; ++k) {
            mma_ss(d, ad + k * astep, b0 + k * (512 >> 4), id, k);
            mma_ss(d + HALF, ad + k * astep, b0 + k * (512 >> 4) + (128 >> 4), id, k);
          }
          mma_commit(&sh.s_full[sb]);
          mma_commit(&sh.empty[sl]);
          if (i == s.n - 1) mma_commit(&sh.q_free[seg & 3]);
          sl += n == 0 ? 1 : 2;
          if (sl >= SLOTS) { sl -= SLOTS; ++round; }
        }
        bar_arrive(&sh.seg_free[seg % SEGS]);
        t += s.n;
      }
      mma_commit(&sh.drained[0]);                                   // (a block that gives up has products on their way)
      bar_drain(smem_u32(&sh.drained[0]), 0);
    }
    __syncwarp();
  } else if (warp == W_PV) {
    // ---- O += P V, behind the clearing of the values behind the unit's last position
    const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(ROWS >> 4) << 24);
    const uint64_t step = page_bytes >> 4;
    uint32_t n = 0, seg = 0, sl = 2, round = 0;      // (V of tile n is use 2 n + 2)
    bool ok = true;
    if (t0 < t1) ok = bar_wait(&sh.full[0], 0, stop);                 // (K0: the one use of slot 0 that is not V's; a wait for V1 would take it for its own)
    for (int t = t0; t < t1 && ok; ++seg) {
      Segment s;
      ok = next_segment(seg, s);
      const uint32_t d = tmem + C_O;
      if (seg > 0) ok = ok && bar_wait(&sh.o_free, seg - 1, stop);
      ok = __all_sync(~0u, ok);
      for (int i = 0; i < s.n && ok; ++i, ++n) {
        const int np = min(PAGES, (s.len + BS - 1) / BS - (s.tile0 + i) * PAGES);
        const uint32_t sb = n % 3, pc = tmem + sb * TP;
        ok = bar_wait(&sh.full[sl], round, stop);
        const int rem = s.len % BS, page = (s.len - 1) / BS - (s.tile0 + i) * PAGES;
        if (ok && rem && page < PAGES) {
          unsigned char* v = base + sl * slot_bytes + page * page_bytes;
          for (int row = lane; row < HD; row += 32) {
            const int sw = (row >> 2) & 1;                            // a row's two 16-byte pieces change places in every other group of four rows
            for (int k = 0; k < 2; ++k) {
              uint4* piece = (uint4*)(v + row * 32 + ((k ^ sw) << 4));
              const int keep = min(8, max(0, rem - 8 * k));
              if (keep == 8) continue;
              uint4 x = *piece;
              uint32_t* e = (uint32_t*)&x;
#pragma unroll
              for (int q = 0; q < 4; ++q) e[q] = 2 * q >= keep ? 0u : 2 * q + 1 >= keep ? e[q] & 0xffffu : e[q];
              *piece = x;
            }
          }
          fence_async();
        }
        ok = ok && bar_wait(&sh.p_full[sb], n / 3, stop);
        ok = __all_sync(~0u, ok);
        if (!ok) break;
        fence_after();
        if (elect()) {
          const uint64_t b = desc(smem_u32(base + sl * slot_bytes), 16, 256, 6);
#pragma unroll 1
          for (int k = 0; k < np; ++k) {
            mma_ts(d, pc + 8 * k, b + k * step, idesc, i + k);
            mma_ts(d, pc + TP / 2 + 8 * k, b + k * step, idesc, 1u);
          }
          mma_commit(&sh.pv_done[sb]);
          mma_commit(&sh.empty[sl]);
          if (i == s.n - 1) mma_commit(&sh.o_full[n & 1]);
        }
        __syncwarp();
        sl += 2;
        if (sl >= SLOTS) { sl -= SLOTS; ++round; }
      }
      if (lane == 0) bar_arrive(&sh.seg_free[seg % SEGS]);
      t += s.n;
    }
    __syncwarp();
    if (elect()) {
      mma_commit(&sh.drained[1]);
      bar_drain(smem_u32(&sh.drained[1]), 0);
    }
    __syncwarp();
  } else if (warp == W_Q) {
    // ---- the segments, and Q: their rows as [HD / 8][rows][8]: 128 rows of a prefix in all of the buffer, a sequence's 16 in one of four places of it
    uint32_t seg = 0, waited = 0;                                   // segments whose rows the products are known to be done with
    const int ch = HD / 8, qn = 32 / ch, qr = lane / ch < qn ? lane / ch : ROWS, qc = lane % ch;
    bool ok = true;
    int own = 0;
    for (int t = t0; t < t1 && ok; ++seg) {
      Segment s;
      segment_at(P, cum, t, t1, s);
      if (seg >= SEGS) ok = __all_sync(~0u, bar_wait(&sh.seg_free[seg % SEGS], seg / SEGS - 1, stop));
      if (lane == 0 && ok) { sh.seg[seg % SEGS] = s; bar_arrive(&sh.seg_full[seg % SEGS]); }
      const uint32_t until = s.own && own ? (seg < 3 ? 0 : seg - 3) : seg;
      for (; waited < until && ok; ++waited) ok = bar_wait(&sh.q_free[waited & 3], waited >> 2, stop);
      ok = __all_sync(~0u, ok);
      if (!ok) break;
      own = s.own;
      const int qrows = s.own ? OWN_ROWS : P.y.qrows;
      const uint32_t dst = smem_u32(qbuf + (s.own ? (seg & 3) * (OWN_ROWS * (uint32_t)HD * 2) : 0u));
      int sq = qr / P.y.G, j = qr - sq * P.y.G;                       // a lane has piece qc of every qn-th row
      for (int row = qr; row < s.rows; row += qn) {
        const __nv_bfloat16* src = (const __nv_bfloat16*)a.q + (s.seq0 + sq) * a.q_stride + (long long)(s.h * P.y.G + j) * HD + qc * 8;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + qc * (qrows * 16) + row * 16), "l"(src) : "memory");
        for (j += qn; j >= P.y.G; j -= P.y.G) ++sq;
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      fence_async();
      bar_arrive(&sh.q_full[seg & 3]);
      t += s.n;
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == W_QK) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  if (tid == 0) {
    P.y.gave_up[worker] = sh.stop;
    if (sh.stop && a.status) atomicOr(a.status, ETXB_SHARED_GAVE_UP);
  }
}

// ------------------------------------------------------------------------------------------------ joining the segments
// A warp has one row: it adds the parts of the prefix's unit and of the sequence's own one, each weighted with 2^(m - M).  Lanes have parts where the weights
// are worked out and four (eight above 128) elements of the output where the parts are added; the order of the sums depends on nothing but the shares.
// What it takes is three trips to L2 behind one another (which workers, their maxima and sums, their results), so each asks for all it can at once.
constexpr int JOIN_THREADS = 128, MAX_WORKERS = 256;
struct JoinParams {                           // (of its own: the first read of every line of a kernel's parameters is a trip to memory)
  const int32_t* prefix_lens; const int32_t* lens; const int32_t* of; const int32_t* gave_up; const int32_t* hdr;
  const float* pO; const float* oO; const float* pml; const float* oml;
  void* out; int32_t* status;
  long long out_stride, pslots;
  int seqs, NH, NKV, HD, G, spt, groups, prows, punits, workers, prefix_max, own_max;          // (positions that the tables have room for)
  Groups first;
};
__global__ void __launch_bounds__(JOIN_THREADS) join_kernel(const __grid_constant__ JoinParams P) {
  const int lane = threadIdx.x & 31, id = blockIdx.x * (JOIN_THREADS / 32) + (threadIdx.x >> 5);
  if (id >= P.seqs * P.NH) return;
  const int HD = P.HD, G = P.G, b = id / P.NH, head = id - b * P.NH, h = head / G, j = head - h * G;
  int g = 0, hi = P.groups - 1;                                     // the group of b: the last that begins at or before it
  while (g < hi) { const int mid = (g + hi + 1) >> 1; if (P.first.first[mid] <= b) g = mid; else hi = mid - 1; }
  const int first = P.first.first[g], um = (b - first) / P.spt, mt = (P.first.first[g + 1] - first + P.spt - 1) / P.spt;
  const int pu = (first / P.spt + g) * P.NKV + h * mt + um, ou = b * P.NKV + h;                 // (see prefix_unit)
  const int size = P.first.first[g + 1] - first, prow = (b - first - um * P.spt) * G + j, prows = min(P.spt, size - um * P.spt) * G;
  const int pl = __ldg(P.prefix_lens + g), ol = __ldg(P.lens + b);
  int2 po = __ldcg((const int2*)P.of + pu), oo = __ldcg((const int2*)P.of + P.punits + ou);
  // where worker 0's parts would be (see part_row): the others' offsets fit 32 bits
  const int pieces = HD / 4, prow0 = (first * P.NKV + h * size + um * P.spt) * G, orow0 = ou * G;
  const float2* const pml = (const float2*)P.pml + prow0 + prow;
  const float2* const oml = (const float2*)P.oml + orow0 + j;
  const float4* const pO = (const float4*)P.pO + (int64_t)prow0 * pieces + prow;
  const float4* const oO = (const float4*)P.oO + (int64_t)orow0 * pieces + j;
  int lost = 0;
#pragma unroll
  for (int w = 0; w < MAX_WORKERS; w += 32) if (w + lane < P.workers) lost |= __ldcg(P.gave_up + w + lane);
  int bad = pl < 0 || pl > P.prefix_max || ol < 0 || ol > P.own_max ? ETXB_SHARED_BAD_LENGTH : 0;
  if (__any_sync(~0u, lost)) bad |= ETXB_SHARED_GAVE_UP;            // (something is unwritten: nothing is looked at)
  const int n0 = bad || pl <= 0 ? 0 : po.y - po.x + 1, n = n0 + (bad || ol <= 0 ? 0 : oo.y - oo.x + 1);
  // part i: the prefix's from worker po.x on, then the own ones
  auto sums = [&](int i) { return __ldcg(i < n0 ? pml + (po.x + i) * P.prows : oml + (oo.x + i - n0) * G); };
  float M = -INFINITY, L = 0.f;
  float2 mine = make_float2(-INFINITY, 0.f);
  for (int i = lane; i < n; i += 32) {
    const float2 s = sums(i);
    bad |= __ldcg(i < n0 ? P.hdr + (pu + po.x + i) : P.hdr + P.pslots + (ou + oo.x + i - n0));
    M = fmaxf(M, s.x);
    if (i < 32) mine = s;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) { M = fmaxf(M, __shfl_xor_sync(~0u, M, o)); bad |= __shfl_xor_sync(~0u, bad, o); }
  const int pstep = P.prows * pieces, ostep = G * pieces;
  float4 y[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
#pragma unroll 1
  for (int i0 = 0; i0 < n; i0 += 32) {
    if (i0 > 0) mine = i0 + lane < n ? sums(i0 + lane) : make_float2(-INFINITY, 0.f);
    // (a part with nothing but scores of minus infinity has no weight; one that is NaN goes on)
    const float w = mine.y == 0.f ? 0.f : mine.x == M ? 1.f : ex2(mine.x - M);
    if (mine.y != 0.f) L = __fmaf_rn(mine.y, w, L);
    const int left = min(32, n - i0);
#pragma unroll 1
    for (int c = 0; c * 32 < pieces; ++c) {
      const int piece = min(c * 32 + lane, pieces - 1);
#pragma unroll 1
      for (int i1 = 0; i1 < left; i1 += 8) {
        float4 v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int i = i0 + min(i1 + k, left - 1);
          v[k] = __ldcg(i < n0 ? pO + ((po.x + i) * pstep + piece * prows) : oO + ((oo.x + i - n0) * ostep + piece * G));
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float wi = __shfl_sync(~0u, w, (i1 + k) & 31);
          if (i1 + k < left && wi != 0.f) {
            float4& z = c ? y[1] : y[0];
            z.x = __fmaf_rn(v[k].x, wi, z.x); z.y = __fmaf_rn(v[k].y, wi, z.y); z.z = __fmaf_rn(v[k].z, wi, z.z); z.w = __fmaf_rn(v[k].w, wi, z.w);
          }
        }
      }
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) L += __shfl_xor_sync(~0u, L, o);
  if (bad && P.status && lane == 0) atomicOr(P.status, bad);
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    if (c * 32 + lane >= pieces) break;
    const float z[4] = {y[c].x / L, y[c].y / L, y[c].z / L, y[c].w / L};
    __nv_bfloat162 out[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) out[e] = __floats2bfloat162_rn(bad ? NAN : L == 0.f ? 0.f : z[2 * e], bad ? NAN : L == 0.f ? 0.f : z[2 * e + 1]);
    *(uint2*)((__nv_bfloat16*)P.out + b * P.out_stride + (int64_t)head * HD + 4 * (c * 32 + lane)) = *(const uint2*)out;
  }
}

// ------------------------------------------------------------------------------------------------ host
static const char* check(const etxb_attn_shared_args& a) {
  if (a.NKV < 1 || a.NH < a.NKV || a.NH % a.NKV || a.NH / a.NKV > 16) return "NH a multiple of NKV, at most 16 q heads per kv head";
  if (a.HD < 16 || a.HD > 256 || a.HD % 16) return "head_dim a multiple of 16, at most 256";
  if (a.seqs < 0 || a.seqs > ETXB_SHARED_MAX_SEQS || a.groups < 0 || a.groups > ETXB_SHARED_MAX_SEQS) return "at most 1024 sequences and groups";
  if (!(a.scale >= 0.f) || a.scale > 1e30f) return "a scale of 0 .. 1e30";
  if (a.pages < 1 || a.table_width < 0 || a.prefix_width < 0 || a.table_width > (1 << 26) || a.prefix_width > (1 << 26)) return "pools of at least one page, tables of at most 2^26 entries a row";
  return nullptr;
}
static const char* check_pointers(const etxb_attn_shared_args& a) {
  if (!a.q || !a.out || !a.kc || !a.vc || !a.lens || !a.prefix_lens || (a.table_width && !a.tables) || (a.prefix_width && !a.prefix_tables) || !a.group_first) return "a pointer is null";
  if (((uintptr_t)a.q | (uintptr_t)a.out | (uintptr_t)a.kc | (uintptr_t)a.vc) & 15) return "q, out and the caches begin at multiples of 16 bytes";
  if (((uintptr_t)a.tables | (uintptr_t)a.lens | (uintptr_t)a.prefix_tables | (uintptr_t)a.prefix_lens | (uintptr_t)a.status) & 3) return "tables and lengths are not aligned to their elements";
  const int64_t row = (int64_t)a.NH * a.HD, page = (int64_t)a.NKV * a.HD * BS;
  if ((a.seqs > 1 && (a.q_stride < row || a.out_stride < row)) || a.q_stride % 8 || a.out_stride % 8) return "rows of q and out lie a multiple of 8 elements apart and do not overlap";
  if (a.k_stride < page || a.v_stride < page || a.k_stride % 8 || a.v_stride % 8) return "pages lie a multiple of 8 elements apart and do not overlap";
  if ((a.seqs > 1 && a.table_stride < a.table_width) || (a.groups > 1 && a.prefix_stride < a.prefix_width)) return "rows of the tables overlap";
  return nullptr;
}
static const char* check_groups(const etxb_attn_shared_args& a) {
  const char* why = "the groups cover the sequences in order";
  if (!a.group_first || a.group_first[0] != 0 || a.group_first[a.groups] != a.seqs) return why;
  for (int g = 0; g < a.groups; ++g) if (a.group_first[g + 1] < a.group_first[g]) return why;
  return nullptr;
}
static int32_t refuse(int32_t code, const char* why) {
  char m[200];
  snprintf(m, sizeof m, "attn_shared: %s", why);
  return etxb_host_fail(code, m);
}


static size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }
// Sizes and places of the partial results from the shapes and the groups; false where the tiles cannot be counted in 31 bits.
static bool lay_out(const etxb_attn_shared_args& a, int workers, unsigned char* work, Layout& y, size_t& bytes) {
  y.G = a.NH / a.NKV; y.spt = ROWS / y.G; y.tp = a.HD <= 128 ? 128 : 64; y.workers = workers;
  int most = 0;
  long long units = 0;
  for (int g = 0; g < a.groups; ++g) {
    const int n = a.group_first[g + 1] - a.group_first[g];
    most = n > most ? n : most;
    units += (n + y.spt - 1) / y.spt;
  }
  const long long tiles = (units * ((a.prefix_width * (long long)BS + y.tp - 1) / y.tp) + a.seqs * ((a.table_width * (long long)BS + y.tp - 1) / y.tp)) * a.NKV;
  if (tiles >= (1ll << 31)) return false;
  y.prows = (most < y.spt ? most : y.spt) * y.G;
  y.punits = (a.seqs / y.spt + a.groups) * a.NKV;
  y.pslots = (long long)y.punits + workers;
  y.oslots = (long long)a.seqs * a.NKV + workers;
  size_t at = 0;
  auto take = [&](size_t n) { unsigned char* p = work + at; at += up256(n); return p; };
  const size_t prows = (size_t)a.seqs * a.NH + (size_t)y.prows * workers;      // (see part_row)
  y.pO = (float*)take(prows * a.HD * 4);
  y.oO = (float*)take((size_t)y.oslots * y.G * a.HD * 4);
  y.pml = (float*)take(prows * 8);
  y.oml = (float*)take((size_t)y.oslots * y.G * 8);
  y.hdr = (int32_t*)take((size_t)(y.pslots + y.oslots) * 4);
  y.gave_up = (int32_t*)take((size_t)workers * 4);
  y.of = (int32_t*)take(((size_t)y.punits + (size_t)a.seqs * a.NKV) * 8);
  bytes = at;
  return true;
}
typedef CUresult (*encode_fn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

}  // namespace etxb_shared

static int32_t sizes(int device, const etxb_attn_shared_args& a, unsigned char* work, etxb_shared::Layout& y, size_t& bytes) {
  using namespace etxb_shared;
  int sms = 0;
  ETXB_HOST_CU(etxb_host_sms(device, &sms));
  if (sms > MAX_WORKERS) sms = MAX_WORKERS;
  if (!lay_out(a, sms, work, y, bytes)) return refuse(ETXB_E_UNSUPPORTED, "the tables' widths allow 2^31 tiles");
  return ETXB_OK;
}

extern "C" int32_t etxb_attn_shared_work(int device, const etxb_attn_shared_args* args, size_t bytes, size_t* work_bytes) {
  using namespace etxb_shared;
  if (!args || bytes != sizeof(etxb_attn_shared_args) || !work_bytes) return refuse(ETXB_E_ARG, "needs an etxb_attn_shared_args");
  if (device < 0 || device >= 64) return refuse(ETXB_E_ARG, "device index out of range");
  if (const char* why = check(*args)) return refuse(ETXB_E_UNSUPPORTED, why);
  *work_bytes = 0;
  if (args->seqs == 0) return ETXB_OK;
  if (const char* why = check_groups(*args)) return refuse(ETXB_E_ARG, why);
  Layout y;
  return sizes(device, *args, nullptr, y, *work_bytes);
}

extern "C" int32_t etxb_attn_shared(int device, const etxb_attn_shared_args* args, size_t bytes, void* cuda_stream) {
  using namespace etxb_shared;
  if (!args || bytes != sizeof(etxb_attn_shared_args)) return refuse(ETXB_E_ARG, "needs an etxb_attn_shared_args");
  if (device < 0 || device >= 64) return refuse(ETXB_E_ARG, "device index out of range");
  if (const char* why = check(*args)) return refuse(ETXB_E_UNSUPPORTED, why);
  if (args->reserved != 0) return refuse(ETXB_E_ARG, "reserved is 0");
  if (args->seqs == 0) return ETXB_OK;
  if (const char* why = check_pointers(*args)) return refuse(ETXB_E_ARG, why);
  if (const char* why = check_groups(*args)) return refuse(ETXB_E_ARG, why);
  EtxbDeviceScope scope(device);
  ETXB_HOST_CU(scope.err);
  static thread_local Params P;                                     // (4 KB of groups: not on a small stack)
  size_t need = 0;
  if (int32_t rc = sizes(device, *args, (unsigned char*)args->work, P.y, need)) return rc;
  if (!args->work || args->work_bytes < need || ((uintptr_t)args->work & 255)) return refuse(ETXB_E_ARG, "work: as many bytes as etxb_attn_shared_work asks for, at a multiple of 256");
  const etxb_attn_shared_args& a = *args;
  P.a = a;
  P.a.group_first = nullptr;
  memset(&P.groups, 0, sizeof P.groups);
  memcpy(P.groups.first, a.group_first, (size_t)(a.groups + 1) * 4);
  static std::atomic<encode_fn> known{nullptr};
  encode_fn encode = known.load(std::memory_order_relaxed);
  if (!encode) {
    cudaDriverEntryPointQueryResult q;
    void* fn = nullptr;
    ETXB_HOST_CU(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q));
    if (!fn || q != cudaDriverEntryPointSuccess) return refuse(ETXB_E_CUDA, "the driver does not offer cuTensorMapEncodeTiled");
    encode = (encode_fn)fn;
    known.store(encode, std::memory_order_relaxed);
  }
  const cuuint64_t dim[3] = {BS, (cuuint64_t)a.NKV * a.HD, (cuuint64_t)a.pages}, str[2] = {BS * 2, (cuuint64_t)a.v_stride * 2};
  const cuuint32_t box[3] = {BS, (cuuint32_t)a.HD, 1}, one[3] = {1, 1, 1};
  const CUresult r = encode(&P.vmap, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, (void*)a.vc, dim, str, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_32B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return refuse(ETXB_E_CUDA, "cuTensorMapEncodeTiled failed for the values");
  const void* k = a.HD > 128 ? (const void*)tiles_kernel<64> : (const void*)tiles_kernel<128>;
  P.y.qrows = P.y.prows <= OWN_ROWS ? OWN_ROWS : (P.y.prows + 7) & ~7;
  const int slot = P.y.tp * a.HD * 2, other = 256 + q_size(a.HD, P.y.qrows) + (a.groups + a.seqs + 1) * 8 + 2048;
  const int slots = (232448 - (int)sizeof(Shared) - 1024 - other) / slot & ~1;
  P.y.slots = slots > MAX_SLOTS ? MAX_SLOTS : slots;                // (four at least: 128 rows of Q and 1024 sequences leave 130 KB)
  static_assert(232448 - (int)sizeof(Shared) - 1024 - (256 + ROWS * 256 * 2 + (2 * ETXB_SHARED_MAX_SEQS + 1) * 8 + 2048) >= 4 * 64 * 256 * 2, "a ring of four tiles");
  const int smem = other + P.y.slots * slot;
  static std::atomic<char> ready[2][64];
  ETXB_HOST_CU(etxb_host_smem(k, 232448 - (int)sizeof(Shared) - 1024, device, ready[a.HD > 128]));
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof cfg);
  cfg.gridDim = dim3((unsigned)P.y.workers); cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = (size_t)smem; cfg.stream = (cudaStream_t)cuda_stream;
  void* kargs[] = {(void*)&P};
  ETXB_HOST_CU(cudaLaunchKernelExC(&cfg, k, kargs));
  static thread_local JoinParams J;
  const Layout& y = P.y;
  J.prefix_lens = a.prefix_lens; J.lens = a.lens; J.of = y.of; J.gave_up = y.gave_up; J.hdr = y.hdr;
  J.pO = y.pO; J.oO = y.oO; J.pml = y.pml; J.oml = y.oml; J.out = a.out; J.status = a.status; J.out_stride = a.out_stride; J.pslots = y.pslots;
  J.seqs = a.seqs; J.NH = a.NH; J.NKV = a.NKV; J.HD = a.HD; J.G = y.G; J.spt = y.spt; J.groups = a.groups; J.prows = y.prows; J.punits = y.punits; J.workers = y.workers;
  J.prefix_max = a.prefix_width * BS; J.own_max = a.table_width * BS;
  J.first = P.groups;
  cfg.gridDim = dim3((unsigned)((a.seqs * a.NH + JOIN_THREADS / 32 - 1) / (JOIN_THREADS / 32))); cfg.blockDim = dim3(JOIN_THREADS); cfg.dynamicSmemBytes = 0;
  void* jargs[] = {(void*)&J};
  ETXB_HOST_CU(cudaLaunchKernelExC(&cfg, (const void*)join_kernel, jargs));
  return ETXB_OK;
}
