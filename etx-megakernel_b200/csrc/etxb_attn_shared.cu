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
// P goes in as two bf16 numbers, P = hi + lo with hi cut off and lo rounded: 16 bits or more.  One would round every probability by 2^-9, which contexts
// of few positions show in the output; the second product is 512 clocks of tensor pipe a tile, beside the 2900 clocks that a tile's bytes take from HBM.
//
// Roles: four warps of softmax; a warp that copies keys and values into a ring of tiles; a thread that issues the products; a warp that fetches the rows of
// the next segment's Q; one that clears the values behind the last position (whatever the cache holds there, 0 times it must be 0).  They meet at mbarriers
// only, so products, softmax and copies of neighbouring tiles and segments overlap: QK of tile n + 1 is issued before PV of tile n, and a segment's results are
// written out while the next one's first products run.  Every wait is bounded.
#include <cuda.h>
#include <cuda_bf16.h>
#include <stdio.h>
#include <string.h>

#include "etxb_host.h"

namespace etxb_shared {

constexpr int BS = 16, ROWS = 128, SLOTS = 4, SLOT_BYTES = 32768;
constexpr int W_COPY = 4, W_MMA = 5, W_Q = 6, THREADS = 256;     // (softmax: 0 .. 3; the last one clears)
constexpr unsigned long long WAIT_NS = 2000000000ull;

struct Groups { int32_t first[ETXB_SHARED_MAX_SEQS + 1]; };

// What both kernels derive alike from the sizes: where a unit's partial results lie.
struct Layout {
  int G, spt;                 // q heads per kv head; sequences whose rows fill a unit of a prefix
  int tp;                     // positions of a tile
  int workers;
  int prows;                  // rows of a slot of a prefix
  long long pslots, oslots;   // slots of prefixes / of own positions
  float* pO; float* pml; float* oO; float* oml;      // [slot][HD / 4][rows][4], [slot][rows][2] (m in units of log2, l)
  int32_t* hdr;               // [pslots + oslots]: status bits of a segment
  int32_t* state;             // [workers]: not 0 where a worker gave up
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
// Waits for phase `n` (0, 1, ..) of a barrier; false, for everyone from then on, when it takes two seconds.
__device__ __forceinline__ bool bar_wait(uint64_t* b, uint32_t n, volatile int* stop) {
  if (bar_try(b, n & 1)) return true;
  const unsigned long long t0 = now_ns();
  for (uint32_t i = 1;; ++i) {
    if (bar_try(b, n & 1)) return true;
    if ((i & 15) == 0) {
      if (*stop) return false;
      if (now_ns() - t0 > WAIT_NS) { *stop = 1; return false; }
    }
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

// ------------------------------------------------------------------------------------------------ shares
// Tiles before group g / sequence b in the order of all tiles: the prefixes' units (group, kv head, rows), then the sequences' (sequence, kv head).
struct Cum {
  int32_t p[ETXB_SHARED_MAX_SEQS + 1], s[ETXB_SHARED_MAX_SEQS + 1];
};
__device__ __forceinline__ bool bad_length(int len, int width) { return len < 0 || len > width * BS; }
__device__ __forceinline__ int tiles_of(int len, int width, int tp) { return bad_length(len, width) ? 0 : (len + tp - 1) / tp; }
__device__ __forceinline__ int units_of(const Params& P, int g) { return (P.groups.first[g + 1] - P.groups.first[g] + P.y.spt - 1) / P.y.spt; }

// Fills c (threads 0 .. 63 of the block; the caller's barrier follows).
__device__ void cumulate(const Params& P, Cum& c) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (warp > 1) return;
  const etxb_attn_shared_args& a = P.a;
  const int n = warp == 0 ? a.groups : a.seqs;
  int32_t* out = warp == 0 ? c.p : c.s;
  int base = 0;
  for (int i0 = 0; i0 < n; i0 += 32) {
    const int i = i0 + lane;
    int v = 0;
    if (i < n) v = warp == 0 ? tiles_of(a.prefix_lens[i], a.prefix_width, P.y.tp) * units_of(P, i) * a.NKV : tiles_of(a.lens[i], a.table_width, P.y.tp) * a.NKV;
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
__device__ __forceinline__ int share(long long total, int w, int workers) { return (int)(total * w / workers); }

struct Segment {
  bool own;
  int who, h;                 // group or sequence; kv head
  int seq0, rows;             // first sequence and number of rows
  int tile0, n;               // tiles [tile0, tile0 + n) of the unit
  int len;                    // positions of the unit
  long long slot;             // of its partial results, prefixes' first
  const int32_t* table;
};
__device__ __forceinline__ Segment segment_at(const Params& P, const Cum& c, int t, int end, int worker) {
  const etxb_attn_shared_args& a = P.a;
  Segment s;
  const int tp_all = c.p[a.groups];
  s.own = t >= tp_all;
  if (!s.own) {
    const int g = s.who = find(c.p, a.groups, t), mt = units_of(P, g), size = P.groups.first[g + 1] - P.groups.first[g];
    const int per = (c.p[g + 1] - c.p[g]) / (mt * a.NKV), rel = t - c.p[g], unit = rel / per;
    s.h = unit / mt;
    const int m = unit - s.h * mt;
    s.seq0 = P.groups.first[g] + m * P.y.spt;
    s.rows = min(P.y.spt, size - m * P.y.spt) * P.y.G;
    s.tile0 = rel - unit * per;
    s.n = min(per - s.tile0, end - t);
    s.len = a.prefix_lens[g];
    s.table = a.prefix_tables + g * a.prefix_stride;
    s.slot = (long long)(P.groups.first[g] / P.y.spt + g) * a.NKV + unit + worker;
  } else {
    const int r = t - tp_all, b = s.who = find(c.s, a.seqs, r);
    const int per = (c.s[b + 1] - c.s[b]) / a.NKV, rel = r - c.s[b];
    s.h = rel / per;
    s.seq0 = b; s.rows = P.y.G;
    s.tile0 = rel - s.h * per;
    s.n = min(per - s.tile0, end - t);
    s.len = a.lens[b];
    s.table = a.tables + b * a.table_stride;
    s.slot = P.y.pslots + (long long)b * a.NKV + s.h + worker;
  }
  return s;
}

// ------------------------------------------------------------------------------------------------ the tiles
struct Shared {
  Cum cum;
  uint64_t full[SLOTS], empty[SLOTS];         // ring of key / value tiles: K0 K1 V0 K2 V1 .. (V of tile n: use 2 n + 2)
  uint64_t v_ready[4];                        // tile n's values are there and those behind the last position cleared, at n % 4 (the ring holds fewer tiles)
  uint64_t s_full[2], p_full[2], pv_done, o_full[2], o_free[2], q_full[2], q_free[2];
  uint32_t tmem;
  int stop;
};

template <int TP>
__global__ void __launch_bounds__(THREADS, 1) tiles_kernel(const __grid_constant__ Params P) {
  extern __shared__ __align__(1024) unsigned char dyn[];
  __shared__ Shared sh;
  constexpr int PAGES = TP / BS, HALF = TP / 2;                     // pages of a tile; columns of S that one half of the pages' positions take
  constexpr int NO = TP == 128 ? 2 : 1, NQ = NO;                    // accumulators of O and buffers of Q: two where they fit
  const etxb_attn_shared_args& a = P.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, HD = a.HD, worker = blockIdx.x;
  const uint32_t page_bytes = (uint32_t)HD * BS * 2, q_bytes = ROWS * (uint32_t)HD * 2;
  unsigned char* const base = (unsigned char*)(((uintptr_t)dyn + 1023) & ~(uintptr_t)1023);
  unsigned char* const qbuf = base + SLOTS * SLOT_BYTES;
  volatile int* const stop = &sh.stop;

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // (what follows on the device waits for this grid before it reads)
  if (tid == 0) {
    for (int i = 0; i < SLOTS; ++i) { bar_init(&sh.full[i], 1); bar_init(&sh.empty[i], 1); }
    bar_init(&sh.pv_done, 1);
    for (int i = 0; i < 4; ++i) bar_init(&sh.v_ready[i], 32);
    for (int i = 0; i < 2; ++i) {
      bar_init(&sh.s_full[i], 1); bar_init(&sh.p_full[i], 4); bar_init(&sh.o_full[i], 1); bar_init(&sh.o_free[i], 4);
      bar_init(&sh.q_full[i], 32); bar_init(&sh.q_free[i], 1);
    }
    sh.stop = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  cumulate(P, sh.cum);
  if (warp == W_MMA) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sh.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    fence_before();
  }
  fence_async();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sh.tmem;
  const Cum& cum = sh.cum;
  const long long total = (long long)cum.p[a.groups] + cum.s[a.seqs];
  const int t0 = share(total, worker, P.y.workers), t1 = share(total, worker + 1, P.y.workers);

  if (warp < 4) {
    // ---- softmax: row = thread
    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    const float sl = a.scale * 1.4426950408889634f;                 // scores in units of log2
    uint32_t n = 0, seg = 0;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    // Results of the segment before, written while the present one's first products run.
    Segment prev = {};
    float prev_m = 0.f, prev_l = 0.f;
    auto write_out = [&](uint32_t sg) {
      const uint32_t ob = sg % NO;
      ok = ok && bar_wait(&sh.o_full[ob], sg / NO, stop);
      ok = __all_sync(~0u, ok);
      fence_after();
      if (ok && warp * 32 < prev.rows) {
        const int stride = prev.own ? P.y.G : P.y.prows;
        const long long slot = prev.own ? prev.slot - P.y.pslots : prev.slot;
        float* O = (prev.own ? P.y.oO : P.y.pO) + slot * stride * HD + (size_t)tid * 4;
        if (tid < prev.rows) {
          float* ml = (prev.own ? P.y.oml : P.y.pml) + (slot * stride + tid) * 2;
          ml[0] = prev_m; ml[1] = prev_l;
        }
        for (int c = 0; c < HD; c += 16) {
          uint32_t r[16];
          tmem_ld16(tmem + lanes + 2 * TP + ob * HD + c, r);
          tmem_wait_ld();
          if (tid < prev.rows) {
#pragma unroll
            for (int k = 0; k < 4; ++k) *(uint4*)(O + (size_t)(c / 4 + k) * stride * 4) = make_uint4(r[4 * k], r[4 * k + 1], r[4 * k + 2], r[4 * k + 3]);
          }
        }
      }
      fence_before();
      __syncwarp();
      if (lane == 0) bar_arrive(&sh.o_free[ob]);
    };
    for (int t = t0; t < t1 && ok;) {
      const Segment s = segment_at(P, cum, t, t1, worker);
      const bool busy = warp * 32 < s.rows;                         // (a warp without rows only keeps the others' time)
      for (int i = 0; i < s.n && ok; ++i, ++n) {
        const uint32_t sb = n & 1, scol = tmem + lanes + sb * TP;
        ok = bar_wait(&sh.s_full[sb], n >> 1, stop);
        ok = __all_sync(~0u, ok);
        if (!ok) break;
        fence_after();
        if (busy) {
          uint32_t r[TP];
#pragma unroll
          for (int c = 0; c < TP; c += 32) tmem_ld32(scol + c, r + c);
          tmem_wait_ld();
          const int valid = s.len - (s.tile0 + i) * TP;
          // column c holds position (c % HALF) / 8 * 16 + c / HALF * 8 + c % 8 of the tile
          if (valid < TP) {
#pragma unroll
            for (int c = 0; c < TP; ++c) if ((c % HALF) / 8 * 16 + c / HALF * 8 + c % 8 >= valid) r[c] = 0xff800000u;
          }
          float mt = -INFINITY;
#pragma unroll
          for (int c = 0; c < TP; c += 2) mt = fmaxf(mt, fmaxf(__uint_as_float(r[c]), __uint_as_float(r[c + 1])));
          if (i == 0) { m = mt; l = 0.f; }
          else {
            // the maximum moves only when the new one is above it by a factor of 2^8 or more: till then probabilities of up to 2^8 do no harm
            const bool up = m != -INFINITY && (mt - m) * sl > 8.f;
            if (__any_sync(~0u, up)) {
              const float f = up ? ex2((m - mt) * sl) : 1.f;
              ok = bar_wait(&sh.pv_done, n - 1, stop);
              ok = __all_sync(~0u, ok);
              if (!ok) break;
              fence_after();
              const uint32_t ocol = tmem + lanes + 2 * TP + (seg % NO) * HD;
              for (int c = 0; c < HD; c += 16) {
                uint32_t o[16];
                tmem_ld16(ocol + c, o);
                tmem_wait_ld();
#pragma unroll
                for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                tmem_st16(ocol + c, o);
              }
              l *= f;
            }
            if (up || m == -INFINITY) m = mt;
          }
          const float ms = m == -INFINITY ? 0.f : m * sl;
          const int left = min(valid, TP);
#pragma unroll
          for (int j = 0; j < TP / 32; ++j) {                       // 32 positions (two pages) at a time: 16 columns of hi, 16 of lo
            uint32_t hi[16], lo[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              float x[2], y[2];
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int pos = 32 * j + 2 * k + e, c = (pos / 8 & 1) * HALF + pos / 16 * 8 + pos % 8;
                const float v = __uint_as_float(r[c]);
                float p = ex2(__fmaf_rn(v, sl, -ms));
                if (valid < TP && pos >= left) p = 0.f;
                l += p;
                // hi: the upper 16 bits; lo: what is left, never 0 where p is not (0 x inf would spoil an infinite value's sum)
                const uint32_t u = p == 0.f ? 0u : __float_as_uint(p) | 1u;
                x[e] = __uint_as_float(u & 0xffff0000u);
                y[e] = __uint_as_float(u) - x[e];
              }
              hi[k] = __byte_perm(__float_as_uint(x[0]), __float_as_uint(x[1]), 0x7632);
              const __nv_bfloat162 b2 = __floats2bfloat162_rn(y[0], y[1]);
              lo[k] = *(const uint32_t*)&b2;
            }
            tmem_st16(scol + 16 * j, hi);
            tmem_st16(scol + TP / 2 + 16 * j, lo);
          }
          tmem_wait_st();
        }
        fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(&sh.p_full[sb]);
        if (i == 0 && seg > 0) write_out(seg - 1);
      }
      prev = s; prev_m = m == -INFINITY ? m : m * sl; prev_l = l;
      ++seg;
      t += s.n;
    }
    if (ok && seg > 0) write_out(seg - 1);
  } else if (warp == W_COPY) {
    // ---- copies: a lane per page
    uint32_t use = 0, filled[SLOTS] = {};                           // running number of ring slots taken; how often each was
    bool ok = true;
    Segment s;
    int t = t0, i = 0;
    auto put = [&](int n_pages, int page, int h, bool values) {
      const uint32_t sl = use % SLOTS, round = use / SLOTS;
      if (round > 0) ok = ok && bar_wait(&sh.empty[sl], round - 1, stop);
      ok = __all_sync(~0u, ok);
      if (!ok) return;
#pragma unroll
      for (int i = 0; i < SLOTS; ++i) if (sl == i) filled[i] = round + 1;
      if (lane == 0) bar_expect(&sh.full[sl], n_pages * page_bytes);
      __syncwarp();
      unsigned char* dst = base + sl * SLOT_BYTES + lane * page_bytes;
      if (lane < n_pages) {
        if (values) tma_load_3d(dst, &P.vmap, h * HD, page, &sh.full[sl]);
        else bulk_load(dst, (const __nv_bfloat16*)a.kc + page * a.k_stride + (long long)h * HD * BS, page_bytes, &sh.full[sl]);
      }
      ++use;
    };
    int bad = 0, vp = 0, vn = 0, vh = 0;                            // the tile whose values follow
    bool have = false;
    while (t < t1 && ok) {
      if (i == 0) s = segment_at(P, cum, t, t1, worker);
      const int pg0 = (s.tile0 + i) * PAGES, np = min(PAGES, (s.len + BS - 1) / BS - pg0);
      int page = lane < np ? s.table[pg0 + lane] : 0;
      const bool off = page < 0 || page >= a.pages;
      if (__any_sync(~0u, off)) { bad = ETXB_SHARED_BAD_PAGE; if (off) page = 0; }
      put(np, page, s.h, false);
      if (have) put(vn, vp, vh, true);
      have = true; vp = page; vn = np; vh = s.h;
      if (++i == s.n) {
        if (lane == 0) P.y.hdr[s.slot] = bad;
        if (bad && lane == 0 && a.status) atomicOr(a.status, bad);
        bad = 0; i = 0; t += s.n;
      }
    }
    ++use;
    if (have && ok) put(vn, vp, vh, true);
    // before the block ends, nothing is on its way into its memory any more (also when it gave up)
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
      const unsigned long long w0 = now_ns();
      while (filled[i] && !bar_try(&sh.full[i], (filled[i] - 1) & 1) && now_ns() - w0 < WAIT_NS) {}
    }
  } else if (warp == W_MMA) {
    // ---- products
    const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(ROWS >> 4) << 24);
    const uint32_t idesc_pv = idesc | ((uint32_t)(HD >> 3) << 17);
    uint32_t use = 0, n = 0, seg = 0;
    bool ok = true;
    int t = t0, i = 0;
    Segment s;
    struct { int np; bool first, last; uint32_t seg; } v = {0, false, false, 0};   // the tile whose PV follows
    bool have = false;
    auto pv = [&]() {
      const uint32_t sl = use % SLOTS, m = n - 1, ob = v.seg % NO;
      ok = ok && bar_wait(&sh.full[sl], use / SLOTS, stop);
      ok = ok && bar_wait(&sh.v_ready[m & 3], m >> 2, stop);
      if (v.first && v.seg >= NO) ok = ok && bar_wait(&sh.o_free[ob], v.seg / NO - 1, stop);
      ok = ok && bar_wait(&sh.p_full[m & 1], m >> 1, stop);
      if (!ok) return;
      fence_after();
      if (elect()) {
        const uint32_t d = tmem + 2 * TP + ob * HD, pc = tmem + (m & 1) * TP;
        uint64_t b = desc(smem_u32(base + sl * SLOT_BYTES), 16, 256, 6);
        for (int k = 0; k < v.np; ++k, b += page_bytes >> 4) {
          mma_ts(d, pc + 8 * k, b, idesc_pv, (!v.first || k > 0) ? 1u : 0u);
          mma_ts(d, pc + TP / 2 + 8 * k, b, idesc_pv, 1u);
        }
        mma_commit(&sh.empty[sl]);
        mma_commit(&sh.pv_done);
        if (v.last) mma_commit(&sh.o_full[ob]);
      }
      __syncwarp();
      ++use;
    };
    while (t < t1 && ok) {
      if (i == 0) {
        s = segment_at(P, cum, t, t1, worker);
        ok = bar_wait(&sh.q_full[seg % NQ], seg / NQ, stop);
      }
      const int np = min(PAGES, (s.len + BS - 1) / BS - (s.tile0 + i) * PAGES);
      const uint32_t sl = use % SLOTS;
      ok = ok && bar_wait(&sh.full[sl], use / SLOTS, stop);
      if (!ok) break;
      fence_after();
      if (elect()) {
        const uint32_t id = idesc | ((uint32_t)((np + 1) & ~1) << 17);               // N = 8 positions of each page, a multiple of 16
        const uint32_t qa = smem_u32(qbuf + (seg % NQ) * q_bytes), ka = smem_u32(base + sl * SLOT_BYTES);
        uint64_t ad = desc(qa, ROWS * 16, 128, 0), b0 = desc(ka, 256, page_bytes, 0);
        for (int k = 0; k < HD / 16; ++k, ad += (2 * ROWS * 16) >> 4, b0 += 512 >> 4) {
          mma_ss(tmem + (n & 1) * TP, ad, b0, id, k > 0 ? 1u : 0u);
          mma_ss(tmem + (n & 1) * TP + HALF, ad, b0 + (128 >> 4), id, k > 0 ? 1u : 0u);
        }
        mma_commit(&sh.empty[sl]);
        mma_commit(&sh.s_full[n & 1]);
        if (i == s.n - 1) mma_commit(&sh.q_free[seg % NQ]);
      }
      __syncwarp();
      ++use;
      if (have) pv();
      have = true;
      v = {np, i == 0, i == s.n - 1, seg};
      ++n;
      if (++i == s.n) { i = 0; t += s.n; ++seg; }
    }
    ++use;
    if (have && ok) pv();
  } else if (warp == W_Q) {
    // ---- Q: the rows of a segment as [HD / 8][128 rows][8]
    uint32_t seg = 0;
    for (int t = t0; t < t1; ++seg) {
      const Segment s = segment_at(P, cum, t, t1, worker);
      const uint32_t qb = seg % NQ;
      if (seg >= NQ && !bar_wait(&sh.q_free[qb], seg / NQ - 1, stop)) break;
      const uint32_t dst = smem_u32(qbuf + qb * q_bytes);
      const int ch = HD / 8;
      for (int x = lane; x < s.rows * ch; x += 32) {
        const int row = x / ch, c = x - row * ch, sq = row / P.y.G, j = row - sq * P.y.G;
        const __nv_bfloat16* src = (const __nv_bfloat16*)a.q + (s.seq0 + sq) * a.q_stride + (long long)(s.h * P.y.G + j) * HD + c * 8;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + c * (ROWS * 16) + row * 16), "l"(src) : "memory");
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      fence_async();
      bar_arrive(&sh.q_full[qb]);
      t += s.n;
    }
  } else {
    // ---- values behind the last position of a unit become 0
    // It looks at every tile of values, in order: a wait that skipped some would take an earlier phase of the slot's barrier for the one it means.
    // Ring order K0 K1 V0 K2 V1 .. (behind the last K a use is left out): V of tile n is use 2 n + 2.
    bool ok = true;
    uint32_t n = 0;
    if (t0 < t1) ok = bar_wait(&sh.full[0], 0, stop);                 // (K0: the one use of slot 0 that is not V's)
    for (int t = t0; t < t1 && ok;) {
      const Segment s = segment_at(P, cum, t, t1, worker);
      for (int i = 0; i < s.n && ok; ++i, ++n) {
        const uint32_t u = 2 * n + 2, sl = u % SLOTS;
        ok = bar_wait(&sh.full[sl], u / SLOTS, stop);
        const int rem = s.len % BS, page = (s.len - 1) / BS - (s.tile0 + i) * PAGES;
        if (ok && rem && page < PAGES) {
          unsigned char* v = base + sl * SLOT_BYTES + page * page_bytes;
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
        bar_arrive(&sh.v_ready[n & 3]);
      }
      t += s.n;
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == W_MMA) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  if (tid == 0) {
    P.y.state[worker] = sh.stop;
    if (sh.stop && a.status) atomicOr(a.status, ETXB_SHARED_GAVE_UP);
  }
}

// ------------------------------------------------------------------------------------------------ joining the segments
// A thread has four output elements of one row: it adds the parts of the prefix's unit and of the sequence's own one, each weighted with 2^(m - M).
constexpr int JOIN_THREADS = 256;
__global__ void __launch_bounds__(JOIN_THREADS) join_kernel(const __grid_constant__ Params P) {
  __shared__ Cum cum;
  const etxb_attn_shared_args& a = P.a;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  cumulate(P, cum);
  __syncthreads();
  const int HD = a.HD, G = P.y.G, W = P.y.workers;
  const long long idx = (long long)blockIdx.x * JOIN_THREADS + threadIdx.x;
  if (idx >= (long long)a.seqs * a.NH * (HD / 4)) return;
  const int j = (int)(idx % G);
  const long long r1 = idx / G;
  const int c = (int)(r1 % (HD / 4));
  const long long r2 = r1 / (HD / 4);
  const int h = (int)(r2 % a.NKV), b = (int)(r2 / a.NKV);
  int lo = 0, hi = a.groups - 1;                                    // the group of b: the last that begins at or before it
  while (lo < hi) { const int mid = (lo + hi + 1) >> 1; if (P.groups.first[mid] <= b) lo = mid; else hi = mid - 1; }
  const int g = lo, first = P.groups.first[g], mt = units_of(P, g), um = (b - first) / P.y.spt;
  const long long total = (long long)cum.p[a.groups] + cum.s[a.seqs];
  int bad = 0;
  if (bad_length(a.prefix_lens[g], a.prefix_width) || bad_length(a.lens[b], a.table_width)) bad = ETXB_SHARED_BAD_LENGTH;
  // the two units: tiles [ta, tb) of all, the slot of worker 0, the rows of a slot and this row
  int ta[2], tb[2], stride[2], row[2];
  long long slot[2];
  {
    const int per = (cum.p[g + 1] - cum.p[g]) / (mt * a.NKV), unit = h * mt + um;
    ta[0] = cum.p[g] + unit * per; tb[0] = ta[0] + per;
    slot[0] = (long long)(first / P.y.spt + g) * a.NKV + unit;
    stride[0] = P.y.prows; row[0] = (b - first - um * P.y.spt) * G + j;
    const int po = (cum.s[b + 1] - cum.s[b]) / a.NKV;
    ta[1] = cum.p[a.groups] + cum.s[b] + h * po; tb[1] = ta[1] + po;
    slot[1] = (long long)b * a.NKV + h;
    stride[1] = G; row[1] = j;
  }
  float M = -INFINITY;
  for (int k = 0; k < 2; ++k) {
    if (ta[k] >= tb[k]) continue;
    int w = (int)((long long)ta[k] * W / total);                    // a worker at or before the first; the shares are rounded down
    while (share(total, w + 1, W) <= ta[k]) ++w;
    for (; w < W && share(total, w, W) < tb[k]; ++w) {
      if (share(total, w, W) == share(total, w + 1, W)) continue;   // (more workers than tiles: an empty share)
      const float* ml = (k ? P.y.oml : P.y.pml) + ((slot[k] + w) * stride[k] + row[k]) * 2;
      M = fmaxf(M, __ldcg(ml));
      bad |= P.y.hdr[(k ? P.y.pslots : 0) + slot[k] + w] | (P.y.state[w] ? ETXB_SHARED_GAVE_UP : 0);
    }
  }
  float L = 0.f, y[4] = {0.f, 0.f, 0.f, 0.f};
  for (int k = 0; k < 2; ++k) {
    if (ta[k] >= tb[k]) continue;
    int w = (int)((long long)ta[k] * W / total);
    while (share(total, w + 1, W) <= ta[k]) ++w;
    for (; w < W && share(total, w, W) < tb[k]; ++w) {
      if (share(total, w, W) == share(total, w + 1, W)) continue;
      const float* ml = (k ? P.y.oml : P.y.pml) + ((slot[k] + w) * stride[k] + row[k]) * 2;
      const float m = __ldcg(ml), l = __ldcg(ml + 1);
      if (l == 0.f) continue;                                       // (nothing but scores of minus infinity; NaN goes on)
      const float f = m == M ? 1.f : ex2(m - M);
      const float4 o = __ldcg((const float4*)((k ? P.y.oO : P.y.pO) + (slot[k] + w) * stride[k] * HD + ((size_t)c * stride[k] + row[k]) * 4));
      L = __fmaf_rn(l, f, L);
      y[0] = __fmaf_rn(o.x, f, y[0]); y[1] = __fmaf_rn(o.y, f, y[1]); y[2] = __fmaf_rn(o.z, f, y[2]); y[3] = __fmaf_rn(o.w, f, y[3]);
    }
  }
  if (bad && a.status && c == 0 && j == 0) atomicOr(a.status, bad);
  __nv_bfloat162 out[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const float z0 = bad ? NAN : L == 0.f ? 0.f : y[2 * e] / L, z1 = bad ? NAN : L == 0.f ? 0.f : y[2 * e + 1] / L;
    out[e] = __floats2bfloat162_rn(z0, z1);
  }
  *(uint2*)((__nv_bfloat16*)a.out + b * a.out_stride + (long long)(h * G + j) * HD + 4 * c) = *(const uint2*)out;
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
  y.pslots = ((long long)a.seqs / y.spt + a.groups) * a.NKV + workers;      // (see segment_at: each group's units begin at (first / spt + g) * NKV)
  y.oslots = (long long)a.seqs * a.NKV + workers;
  size_t at = 0;
  auto take = [&](size_t n) { unsigned char* p = work + at; at += up256(n); return p; };
  y.pO = (float*)take((size_t)y.pslots * y.prows * a.HD * 4);
  y.oO = (float*)take((size_t)y.oslots * y.G * a.HD * 4);
  y.pml = (float*)take((size_t)y.pslots * y.prows * 8);
  y.oml = (float*)take((size_t)y.oslots * y.G * 8);
  y.hdr = (int32_t*)take((size_t)(y.pslots + y.oslots) * 4);
  y.state = (int32_t*)take((size_t)workers * 4);
  bytes = at;
  return true;
}
typedef CUresult (*encode_fn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

}  // namespace etxb_shared

static int32_t sizes(int device, const etxb_attn_shared_args& a, unsigned char* work, etxb_shared::Layout& y, size_t& bytes) {
  using namespace etxb_shared;
  int sms = 0;
  ETXB_HOST_CU(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
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
  static encode_fn encode = nullptr;
  if (!encode) {
    cudaDriverEntryPointQueryResult q;
    void* fn = nullptr;
    ETXB_HOST_CU(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q));
    if (!fn || q != cudaDriverEntryPointSuccess) return refuse(ETXB_E_CUDA, "the driver does not offer cuTensorMapEncodeTiled");
    encode = (encode_fn)fn;
  }
  const cuuint64_t dim[3] = {BS, (cuuint64_t)a.NKV * a.HD, (cuuint64_t)a.pages}, str[2] = {BS * 2, (cuuint64_t)a.v_stride * 2};
  const cuuint32_t box[3] = {BS, (cuuint32_t)a.HD, 1}, one[3] = {1, 1, 1};
  const CUresult r = encode(&P.vmap, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, (void*)a.vc, dim, str, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_32B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return refuse(ETXB_E_CUDA, "cuTensorMapEncodeTiled failed for the values");
  const void* k = a.HD <= 128 ? (const void*)tiles_kernel<128> : (const void*)tiles_kernel<64>;
  const int smem = 1024 + SLOTS * SLOT_BYTES + (a.HD <= 128 ? 2 : 1) * ROWS * a.HD * 2;
  ETXB_HOST_CU(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof cfg);
  cfg.gridDim = dim3((unsigned)P.y.workers); cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = (size_t)smem; cfg.stream = (cudaStream_t)cuda_stream;
  void* kargs[] = {(void*)&P};
  ETXB_HOST_CU(cudaLaunchKernelExC(&cfg, k, kargs));
  const long long threads = (long long)a.seqs * a.NH * (a.HD / 4);
  cfg.gridDim = dim3((unsigned)((threads + JOIN_THREADS - 1) / JOIN_THREADS)); cfg.blockDim = dim3(JOIN_THREADS); cfg.dynamicSmemBytes = 0;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at; cfg.numAttrs = 1;
  ETXB_HOST_CU(cudaLaunchKernelExC(&cfg, (const void*)join_kernel, kargs));
  return ETXB_OK;
}
