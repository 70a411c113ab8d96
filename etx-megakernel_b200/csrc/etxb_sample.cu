// Drawing tokens: temperature, top-k, top-p and min-p over rows of logits, with given random numbers (etxb_sample).
//
// Mathematics.  The live tokens of a row (neither -inf nor NaN) stand in the order "larger logit first, equal logits by index".  Token r of that order
// has the weight w_r = exp((l_r - l_0) / T).  Every cut keeps a beginning of the order:
//   top-k   the first min(k, live)                                          mass W_k = the sum of their weights
//   top-p   those with (sum of the weights before r) < p * W_k
//   min-p   those with w_r >= min_p
// so together they keep the first n (at least one).  Drawn is the first token whose inclusive sum exceeds u * W_n.
//
// The sums have to be right next to every border, and the order of atomics must not change them.
//
// Logits of 16 bits (counts_kernel).  A row has at most 65536 different values, and a real one some thousands: the row is counted value by value, exactly, with
// 16-bit counters in shared memory, and then one exp in 64 bits per value that occurs, and sums over values in their order, give all three cuts and the
// draw.  Nothing is sorted.  A row belongs to a cluster of C blocks, each of which counts a part of it; values are joined through distributed shared
// memory, 32 neighbouring ones (a group) at a time, and only groups that occur.
// Logits of 32 bits (sums_kernel).  Bins by the first 11 bits of the value, then the next 11 and the last 10 of one bin: three passes for a border.  A bin has a
// number of tokens and a sum of weights, which are integers: exp in 64 bits times 2^S with S = 62 - ceil(log2 V), so that a row's sum fits 63 bits, is
// exact whatever the order, and a weight is off by 2^-(S+1) <= 2^-43 of the largest.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdio.h>
#include <string.h>

#include "etxb_host.h"

namespace etxb_draw {
namespace cg = cooperative_groups;

constexpr int THREADS = 1024, WARPS = THREADS / 32, MAX_CLUSTER = 8;

// A row's settings, in the form the kernels use.
struct Settings {
  float T, top_p, min_p;
  int k;
  double u;
};
__device__ __forceinline__ Settings settings(const etxb_sample_args& a, int row) {
  Settings s;
  s.T = a.temperature ? a.temperature[row] : a.temperature_all;
  s.k = a.top_k ? a.top_k[row] : a.top_k_all;
  s.top_p = a.top_p ? a.top_p[row] : a.top_p_all;
  s.min_p = a.min_p ? a.min_p[row] : a.min_p_all;
  const float u = a.u[row];
  s.u = u > 0.f ? fmin((double)u, 1.0 - 0x1p-24) : 0.0;
  return s;
}
__device__ __forceinline__ void store(const etxb_sample_args& a, int row, int token, float logp, int kept) {
  a.tokens[row] = token;
  if (a.next) a.next[row] = token;
  if (a.logprobs) a.logprobs[row] = logp;
  if (a.kept) a.kept[row] = kept;
}

// What a lookup asks for: the token of a rank; the last token with less than `x` before it; the first with more than `x` up to it.
enum { BY_RANK, BY_MASS_BEFORE, BY_MASS_UPTO };
template <typename M>
__device__ __forceinline__ bool falls(int how, uint32_t rank, double x, uint32_t c0, uint32_t c, M m0, M m1) {
  if (how == BY_RANK) return c0 <= rank && rank < c0 + c;
  if (how == BY_MASS_BEFORE) return c > 0u && (double)m0 < x && (double)m1 >= x;
  return (double)m0 <= x && (double)m1 > x;
}

// ================================================================================================ logits of 16 bits
// Keys: values as unsigned numbers in the values' order; 0 for -inf and NaN; -0 is +0.  INF: the key of +inf (bf16 0x7f80, fp16 0x7c00).
template <uint32_t INF>
struct Key16 {
  static constexpr uint32_t LOWEST = (uint32_t)(0xffffu - (INF - 1u + 0x8000u)) & 0xffffu;         // the key of the type's lowest number
  static __device__ __forceinline__ uint32_t of(uint32_t u) {                                       // u: 16 bits
    uint32_t k = (u & 0x8000u) ? (~u & 0xffffu) : (u | 0x8000u);
    if (k == 0x7fffu) k = 0x8000u;
    return k - LOWEST <= INF + 0x8000u - LOWEST ? k : 0u;
  }
};
template <typename T> __device__ __forceinline__ float value16(uint32_t key);
template <> __device__ __forceinline__ float value16<__nv_bfloat16>(uint32_t key) {
  return __uint_as_float(((key & 0x8000u) ? (key & 0x7fffu) : (~key & 0xffffu)) << 16);
}
template <> __device__ __forceinline__ float value16<__half>(uint32_t key) {
  return __half2float(__ushort_as_half((unsigned short)((key & 0x8000u) ? (key & 0x7fffu) : (~key & 0xffffu))));
}

constexpr int GROUPS = 2048, CHUNK = 8191;                          // groups of 32 values; vectors of 8 logits a block counts (16 bits hold their number)
struct Counts {
  uint32_t hist[32768];                                             // two counters a word
  double mass[GROUPS], mass_min[GROUPS];                            // of the groups this block joins (a C-th of them): sum of weights, and of those min-p keeps
  uint32_t count[GROUPS], count_min[GROUPS];
  uint16_t list[GROUPS];                                            // of these, the ones that occur
  uint32_t bits[GROUPS / 32];                                       // the groups that occur in this block's part
  uint32_t wc[WARPS], wcm[WARPS];
  double wm[WARPS], wmm[WARPS];
  uint32_t maxkey, n_list;
  uint32_t hit_group, hit_count, place_key, place_before, place_count;
  double hit_mass, place_mass, place_weight;
  int found;
  uint32_t entry, entry_before;
};

template <typename T, int NV>
__global__ void __launch_bounds__(THREADS, 1) counts_kernel(const etxb_sample_args a) {
  using K = Key16<sizeof(T) == 2 && __is_same(T, __half) ? 0x7c00u : 0x7f80u>;
  extern __shared__ __align__(16) unsigned char smem[];
  Counts& s = *(Counts*)smem;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), r = (int)cluster.block_rank(), row = blockIdx.x / C;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = a.V;
  const Settings st = settings(a, row);
  const bool greedy = !(st.T > 0.f);

  // this block's vectors of 8 logits, from the last 16-byte boundary before the row on: logit v * 8 - shift + j
  const T* l = (const T*)a.logits + (long long)row * a.row_stride;
  const int shift = (int)((uintptr_t)l & 15) / 2, nvec = (shift + V + 7) / 8;
  const int v0 = (int)((long long)nvec * r / C), v1 = (int)((long long)nvec * (r + 1) / C);
  uint4 key[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = v0 + i * THREADS + tid;
    key[i] = make_uint4(0u, 0u, 0u, 0u);
    const int e = v * 8 - shift;
    if (v < v1 && e >= 0 && e + 8 <= V) key[i] = __ldg((const uint4*)(l + e));
    else if (v < v1) {                                              // the row's ends, one by one (0xffff is no number)
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int x = e + 2 * j;
        const uint32_t lo = x >= 0 && x < V ? ((const unsigned short*)l)[x] : 0xffffu, hi = x + 1 >= 0 && x + 1 < V ? ((const unsigned short*)l)[x + 1] : 0xffffu;
        w[j] = lo | (hi << 16);
      }
      key[i] = make_uint4(w[0], w[1], w[2], w[3]);
    } else key[i] = make_uint4(~0u, ~0u, ~0u, ~0u);
  }
  if (!greedy)
    for (int i = tid; i < 32768 / 4; i += THREADS) ((uint4*)s.hist)[i] = make_uint4(0u, 0u, 0u, 0u);
  for (int i = tid; i < GROUPS / C; i += THREADS) { s.mass[i] = 0.0; s.mass_min[i] = 0.0; s.count[i] = 0u; s.count_min[i] = 0u; }
  if (tid == 0) { s.maxkey = 0u; s.n_list = 0u; }
  __syncthreads();
  uint32_t mx = 0u, low = 0u;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    uint32_t* w = (uint32_t*)&key[i];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t k0 = K::of(w[j] & 0xffffu), k1 = K::of(w[j] >> 16);
      w[j] = k0 | (k1 << 16);
      mx = max(mx, max(k0, k1));
      if (!greedy) {
        // (a mask of the type's lowest number makes most of a row equal: those are counted without memory)
        if (k0 == K::LOWEST) ++low; else if (k0) atomicAdd(&s.hist[k0 >> 1], 1u << ((k0 & 1u) * 16u));
        if (k1 == K::LOWEST) ++low; else if (k1) atomicAdd(&s.hist[k1 >> 1], 1u << ((k1 & 1u) * 16u));
      }
    }
  }
  mx = __reduce_max_sync(~0u, mx); low = __reduce_add_sync(~0u, low);
  if (lane == 0) { atomicMax(&s.maxkey, mx); if (low) atomicAdd(&s.hist[K::LOWEST >> 1], low << ((K::LOWEST & 1u) * 16u)); }
  __syncthreads();
  if (!greedy) {
    // groups that occur: four lanes look at the 64 bytes of one
    for (int i = 0; i < GROUPS * 4 / THREADS; ++i) {
      const uint4 q = ((const uint4*)s.hist)[i * THREADS + tid];
      uint32_t any = q.x | q.y | q.z | q.w;
      any |= __shfl_xor_sync(~0u, any, 1); any |= __shfl_xor_sync(~0u, any, 2);
      uint32_t b = __ballot_sync(~0u, any != 0u);                   // 8 groups, a nibble each
      if (lane == 0) {
        b &= 0x11111111u;
        b = (b | b >> 3) & 0x03030303u; b = (b | b >> 6) & 0x000f000fu; b = (b | b >> 12) & 0xffu;
        ((unsigned char*)s.bits)[i * (THREADS / 32) + warp] = (unsigned char)b;
      }
    }
  }
  cluster.sync();
  uint32_t maxkey = 0u;
  int first_with_max = 0;
  for (int c = C - 1; c >= 0; --c) {
    const uint32_t m = *cluster.map_shared_rank(&s.maxkey, c);
    if (m >= maxkey) { maxkey = m; first_with_max = c; }
  }
  if (maxkey == 0u) {                                               // nothing is allowed
    if (r == 0 && tid == 0) store(a, row, -1, -INFINITY, 0);
    cluster.sync();
    return;
  }
  const double dmax = (double)value16<T>(maxkey), inv_t = 1.0 / (double)st.T;
  auto log_weight = [&](uint32_t k) { const double d = (double)value16<T>(k) - dmax; return d == d ? d * inv_t : 0.0; };      // (inf - inf: the largest itself)
  auto weight = [&](uint32_t k) { const double d = (double)value16<T>(k) - dmax; return d < 0.0 ? (d == -INFINITY ? 0.0 : exp(d * inv_t)) : 1.0; };
  // tokens of value k in the whole row
  auto tokens_of = [&](uint32_t k) {
    uint32_t n = 0u;
    for (int c = 0; c < C; ++c) n += ((const uint16_t*)cluster.map_shared_rank(&s.hist[0], c))[k];
    return n;
  };

  uint32_t nth = 0u, at = maxkey;                                   // the drawn token: the nth one, by index, of the value `at`
  int kept = 1;
  float logp = 0.f;
  if (!greedy) {
    // this block joins the groups [g0, g0 + GROUPS / C): the list of those that occur, then a warp a group
    const int per = GROUPS / C, g0 = r * per;
    if (tid < per / 32) {
      uint32_t b = 0u;
      for (int c = 0; c < C; ++c) b |= cluster.map_shared_rank(&s.bits[0], c)[g0 / 32 + tid];
      uint32_t n = atomicAdd(&s.n_list, (uint32_t)__popc(b));
      for (; b; b &= b - 1u) s.list[n++] = (uint16_t)(tid * 32 + __ffs(b) - 1);
    }
    __syncthreads();
    for (uint32_t i = warp; i < s.n_list; i += WARPS) {
      const uint32_t g = s.list[i], k = (uint32_t)(g0 + g) * 32u + 31u - (uint32_t)lane;           // lanes from the group's largest value down
      const uint32_t n = tokens_of(k);
      const double w = n ? weight(k) : 0.0;
      const bool in = n && w >= (double)st.min_p;
      double m = (double)n * w, mm = in ? m : 0.0;
#pragma unroll
      for (int o = 16; o; o >>= 1) { m += __shfl_xor_sync(~0u, m, o); mm += __shfl_xor_sync(~0u, mm, o); }
      const uint32_t c = __reduce_add_sync(~0u, n), cm = __reduce_add_sync(~0u, in ? n : 0u);
      if (lane == 0) { s.mass[g] = m; s.mass_min[g] = mm; s.count[g] = c; s.count_min[g] = cm; }
    }
    cluster.sync();
    // every block goes over all groups in descending order, two a thread: tokens and mass before each
    uint32_t gc[2], gb, cm = 0u, total = 0u, total_min = 0u;
    double gm[2], mb, mm = 0.0, total_m = 0.0, total_mm = 0.0;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int g = GROUPS - 1 - (2 * tid + k), c = g / per, x = g - c * per;
      const Counts* o = cluster.map_shared_rank(&s, c);
      gc[k] = o->count[x]; gm[k] = o->mass[x];
      cm += o->count_min[x]; mm += o->mass_min[x];
    }
    gb = gc[0] + gc[1]; mb = gm[0] + gm[1];
    const uint32_t own_c = gb;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t x = __shfl_up_sync(~0u, gb, o);
      const double y = __shfl_up_sync(~0u, mb, o);
      if (lane >= o) { gb += x; mb += y; }
    }
    cm = __reduce_add_sync(~0u, cm);
#pragma unroll
    for (int o = 16; o; o >>= 1) mm += __shfl_xor_sync(~0u, mm, o);
    if (lane == 31) { s.wc[warp] = gb; s.wm[warp] = mb; s.wcm[warp] = cm; s.wmm[warp] = mm; }
    __syncthreads();
    double me;                                                      // mass up to and with this thread's groups
    gb -= own_c;
    {
      const double before = __shfl_up_sync(~0u, mb, 1);
      // the warps' sums in order: each lane one of them
      uint32_t c = s.wc[lane];
      double m = s.wm[lane], mmin = s.wmm[lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(~0u, c, o);
        const double y = __shfl_up_sync(~0u, m, o);
        if (lane >= o) { c += x; m += y; }
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) mmin += __shfl_xor_sync(~0u, mmin, o);
      total = __shfl_sync(~0u, c, 31); total_m = __shfl_sync(~0u, m, 31); total_mm = mmin;
      total_min = __reduce_add_sync(~0u, s.wcm[lane]);
      const uint32_t cw = __shfl_sync(~0u, c, (warp + 31) & 31);
      const double mw = __shfl_sync(~0u, m, (warp + 31) & 31), here = warp ? mw : 0.0, next = __shfl_sync(~0u, m, warp);
      gb += warp ? cw : 0u;
      me = lane < 31 ? mb + here : next;
      mb = lane ? before + here : here;
    }
    // a border: the thread whose group it falls into names it, and a warp goes over the group's values
    auto lookup = [&](int how, uint32_t rank, double x) {
      __syncthreads();
      if (tid == 0) s.found = 0;
      __syncthreads();
      uint32_t c0 = gb;
      double m0 = mb;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const double m1 = k == 0 ? fmin(mb + gm[0], me) : me;       // (what a group ends with is, to the bit, what the next one begins with)
        if (gc[k] && falls(how, rank, x, c0, gc[k], m0, m1)) { s.hit_group = (uint32_t)(GROUPS - 1 - (2 * tid + k)); s.hit_count = c0; s.hit_mass = m0; s.found = 1; }
        c0 += gc[k]; m0 = m1;
      }
      __syncthreads();
      if (s.found && warp == 0) {
        const uint32_t k = s.hit_group * 32u + 31u - (uint32_t)lane, n = tokens_of(k);
        const double w = n ? weight(k) : 0.0;
        uint32_t c = n;
        double m = (double)n * w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t x1 = __shfl_up_sync(~0u, c, o);
          const double y1 = __shfl_up_sync(~0u, m, o);
          if (lane >= o) { c += x1; m += y1; }
        }
        uint32_t cb = __shfl_up_sync(~0u, c, 1);
        double mbef = __shfl_up_sync(~0u, m, 1);
        if (lane == 0) { cb = 0u; mbef = 0.0; }
        cb += s.hit_count;
        const double m0 = s.hit_mass + mbef, m1 = s.hit_mass + m;
        uint32_t hits = __ballot_sync(~0u, n && falls(how, rank, x, cb, n, m0, m1));
        // (sums within a group are rounded apart from the group's: a border on its very end belongs to its last value)
        if (!hits) { const uint32_t some = __ballot_sync(~0u, n != 0u); hits = 1u << (31 - __clz(some)); }
        if (lane == __ffs(hits) - 1) { s.place_key = k; s.place_before = cb; s.place_count = n; s.place_mass = m0; s.place_weight = w; }
      }
      __syncthreads();
      return s.found != 0;
    };
    uint32_t n = total;
    double Wn = total_m;
    if (st.k > 0 && (uint32_t)st.k < total) {
      lookup(BY_RANK, (uint32_t)st.k - 1u, 0.0);
      n = (uint32_t)st.k;
      Wn = s.place_mass + (double)(n - s.place_before) * s.place_weight;
    }
    if (st.top_p < 1.f) {
      const double x = (double)st.top_p * Wn;
      uint32_t np = 1u;
      double Wp = 1.0;
      if (x > 0.0 && lookup(BY_MASS_BEFORE, 0u, x)) {
        const double q = ceil((x - s.place_mass) / s.place_weight);
        const uint32_t in = (uint32_t)fmin(fmax(q, 1.0), (double)s.place_count);
        np = s.place_before + in; Wp = s.place_mass + (double)in * s.place_weight;
      }
      if (np < n) { n = np; Wn = Wp; }
    }
    if (st.min_p > 0.f && total_min < n) {
      n = total_min ? total_min : 1u;
      Wn = total_min ? total_mm : 1.0;
    }
    const double x = st.u * Wn;
    const bool found = lookup(BY_MASS_UPTO, 0u, x);
    if (found) nth = (uint32_t)fmin(fmax(floor((x - s.place_mass) / s.place_weight), 0.0), (double)(s.place_count - 1u));
    if (!found || s.place_before + nth >= n) {                      // rounding next to the last border: the last token that is kept
      lookup(BY_RANK, n - 1u, 0.0);
      nth = n - 1u - s.place_before;
    }
    at = s.place_key;
    logp = (float)(log_weight(at) - log(Wn));
    kept = (int)n;
  }
  // which block has it: the tokens of that value in the blocks before
  bool mine;
  if (greedy) mine = r == first_with_max;
  else {
    uint32_t before = 0u, here = 0u;
    for (int c = 0; c <= r; ++c) { before += here; here = ((const uint16_t*)cluster.map_shared_rank(&s.hist[0], c))[at]; }
    mine = before <= nth && nth < before + here;
    nth -= before;
  }
  if (mine) {
    uint32_t* cnt = (uint32_t*)s.list;                              // matches by vector number and warp: the order of the indices
    uint32_t match[NV];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t* w = (const uint32_t*)&key[i];
      match[i] = 0u;
#pragma unroll
      for (int j = 0; j < 4; ++j) match[i] |= ((w[j] & 0xffffu) == at ? 1u << (2 * j) : 0u) | ((w[j] >> 16) == at ? 2u << (2 * j) : 0u);
      const uint32_t c = __reduce_add_sync(~0u, (uint32_t)__popc(match[i]));
      if (lane == 0) cnt[i * WARPS + warp] = c;
    }
    __syncthreads();
    if (warp == 0) {
      uint32_t c = 0u;
#pragma unroll
      for (int q = 0; q < NV; ++q) c += cnt[lane * NV + q];
      uint32_t before = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const uint32_t x = __shfl_up_sync(~0u, before, o); if (lane >= o) before += x; }
      before -= c;
      if (before <= nth && nth < before + c) {
        int q = 0;
        while (before + cnt[lane * NV + q] <= nth) before += cnt[lane * NV + q++];
        s.entry = (uint32_t)(lane * NV + q); s.entry_before = before;
      }
    }
    __syncthreads();
    if ((int)(s.entry & (WARPS - 1)) == warp) {
      const int i = (int)(s.entry / WARPS);
      uint32_t m = 0u;
#pragma unroll
      for (int q = 0; q < NV; ++q) if (q == i) m = match[q];
      const uint32_t c = (uint32_t)__popc(m), want = nth - s.entry_before;
      uint32_t before = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const uint32_t x = __shfl_up_sync(~0u, before, o); if (lane >= o) before += x; }
      before -= c;
      if (before <= want && want < before + c) {
        for (uint32_t q = before; q < want; ++q) m &= m - 1u;
        store(a, row, (v0 + i * THREADS + tid) * 8 - shift + __ffs(m) - 1, logp, kept);
      }
    }
  }
  cluster.sync();                                                   // (no block leaves while another one reads its counters)
}

// ================================================================================================ logits of 32 bits
constexpr int BINS = 2048;
// Logits as keys whose order as unsigned numbers is the order of the values; 0: not live (-inf, NaN).  -0 counts as +0.
__device__ __forceinline__ uint32_t key_of(float l) {
  uint32_t u = __float_as_uint(l);
  if ((u << 1) > 0xff000000u || u == 0xff800000u) return 0u;
  if ((u << 1) == 0u) u = 0u;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key); }

__device__ __forceinline__ float load(const float* p, int i) { return p[i]; }
__device__ __forceinline__ float load(const __nv_bfloat16* p, int i) { return __bfloat162float(p[i]); }
__device__ __forceinline__ float load(const __half* p, int i) { return __half2float(p[i]); }

struct Bins {
  uint32_t count[BINS], lo[BINS], hi[BINS];
};
struct Shared {
  Bins top, sub;                              // by the first 11 bits of the key; by the next ones of one of those bins
  uint32_t wc[WARPS];
  unsigned long long wm[WARPS];
  uint32_t bin, before_count, count, maxkey, live, kept_min;
  unsigned long long before_mass, mass_min;
  int token;
};

// (a, b) -> sums over the threads before this one, and over all
__device__ void block_scan(Shared& s, uint32_t c, unsigned long long m, uint32_t& cb, unsigned long long& mb, uint32_t& ct, unsigned long long& mt) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t ci = c;
  unsigned long long mi = m;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t co = __shfl_up_sync(~0u, ci, o);
    const unsigned long long mo = __shfl_up_sync(~0u, mi, o);
    if (lane >= o) { ci += co; mi += mo; }
  }
  __syncthreads();
  if (lane == 31) { s.wc[warp] = ci; s.wm[warp] = mi; }
  __syncthreads();
  cb = ci - c; mb = mi - m; ct = 0; mt = 0;
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) { cb += s.wc[w]; mb += s.wm[w]; }
    ct += s.wc[w]; mt += s.wm[w];
  }
}

struct Row {
  double max, inv_t;
  double scale;                               // 2^S
};
__device__ __forceinline__ double log_weight(const Row& r, uint32_t key) {
  const double d = (double)value_of(key) - r.max;
  return d == d ? d * r.inv_t : 0.0;          // (inf - inf: the largest itself)
}
__device__ __forceinline__ double real_weight(const Row& r, uint32_t key) {
  const double d = (double)value_of(key) - r.max;
  return d < 0.0 ? (d == -INFINITY ? 0.0 : exp(d * r.inv_t)) : 1.0;     // (beside an infinite logit a finite one has none, at any temperature)
}
__device__ __forceinline__ unsigned long long weight(const Row& r, uint32_t key) { return __double2ull_rn(real_weight(r, key) * r.scale); }
__device__ __forceinline__ void add(Bins& b, uint32_t i, unsigned long long w) {
  atomicAdd(&b.count[i], 1u);
  const uint32_t lo = (uint32_t)w;
  uint32_t hi = (uint32_t)(w >> 32);
  if (lo) { const uint32_t old = atomicAdd(&b.lo[i], lo); hi += (old + lo < old) ? 1u : 0u; }
  if (hi) atomicAdd(&b.hi[i], hi);
}
__device__ __forceinline__ unsigned long long mass(const Bins& b, int i) { return ((unsigned long long)b.hi[i] << 32) | b.lo[i]; }

struct Place {
  uint32_t key, before_count, count;          // a value, the tokens before its first one, its tokens
  unsigned long long before_mass;
  bool found;
};

// The bin (in descending order) that a lookup falls into, given the tokens and mass before all of them.
__device__ bool find_bin(Shared& s, const Bins& b, int nbins, int how, uint32_t rank, double x, uint32_t c0, unsigned long long m0) {
  const int t = threadIdx.x;
  uint32_t c[2];
  unsigned long long m[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int i = nbins - 1 - (2 * t + k);
    c[k] = i >= 0 ? b.count[i] : 0u; m[k] = i >= 0 ? mass(b, i) : 0ull;
  }
  uint32_t cb, ct;
  unsigned long long mb, mt;
  block_scan(s, c[0] + c[1], m[0] + m[1], cb, mb, ct, mt);
  if (t == 0) s.bin = ~0u;
  __syncthreads();
  cb += c0; mb += m0;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (falls(how, rank, x, cb, c[k], mb, mb + m[k])) { s.bin = (uint32_t)(nbins - 1 - (2 * t + k)); s.before_count = cb; s.before_mass = mb; s.count = c[k]; }
    cb += c[k]; mb += m[k];
  }
  __syncthreads();
  return s.bin != ~0u;
}

template <typename T>
__device__ Place lookup(Shared& s, const T* l, int V, const Row& r, int how, uint32_t rank, double x) {
  Place p;
  p.found = find_bin(s, s.top, BINS, how, rank, x, 0u, 0ull);
  if (!p.found) return p;
  uint32_t prefix = s.bin, cb = s.before_count, n = s.count;
  unsigned long long mb = s.before_mass;
  for (int level = 1; level < 3; ++level) {
    const int bits = level == 1 ? 11 : 10, shift = level == 1 ? 10 : 0, nb = 1 << bits;
    __syncthreads();
    for (int i = threadIdx.x; i < nb; i += THREADS) { s.sub.count[i] = 0u; s.sub.lo[i] = 0u; s.sub.hi[i] = 0u; }
    __syncthreads();
    for (int i = threadIdx.x; i < V; i += THREADS) {
      const uint32_t k = key_of(load(l, i));
      if (k && (k >> (shift + bits)) == prefix) add(s.sub, (k >> shift) & (nb - 1), weight(r, k));
    }
    __syncthreads();
    p.found = find_bin(s, s.sub, nb, how, rank, x, cb, mb);
    if (!p.found) return p;                   // (cannot be: the sums of a bin are the bin's)
    prefix = (prefix << bits) | s.bin; cb = s.before_count; mb = s.before_mass; n = s.count;
  }
  p.key = prefix; p.before_count = cb; p.before_mass = mb; p.count = n;
  return p;
}

template <typename T>
__global__ void __launch_bounds__(THREADS) rows_kernel(const etxb_sample_args a) {
  extern __shared__ __align__(16) unsigned char smem[];
  Shared& s = *(Shared*)smem;
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 31, V = a.V;
  const T* l = (const T*)a.logits + (long long)row * a.row_stride;
  const float Tm = a.temperature ? a.temperature[row] : a.temperature_all;
  const int k = a.top_k ? a.top_k[row] : a.top_k_all;
  const float top_p = a.top_p ? a.top_p[row] : a.top_p_all, min_p = a.min_p ? a.min_p[row] : a.min_p_all;

  if (tid == 0) { s.maxkey = 0u; s.live = 0u; s.kept_min = 0u; s.mass_min = 0ull; s.token = -1; }
  for (int i = tid; i < BINS; i += THREADS) { s.top.count[i] = 0u; s.top.lo[i] = 0u; s.top.hi[i] = 0u; }
  __syncthreads();
  uint32_t mx = 0u, live = 0u;
  for (int i = tid; i < V; i += THREADS) { const uint32_t key = key_of(load(l, i)); mx = max(mx, key); live += key ? 1u : 0u; }
  mx = __reduce_max_sync(~0u, mx); live = __reduce_add_sync(~0u, live);
  if (lane == 0) { atomicMax(&s.maxkey, mx); atomicAdd(&s.live, live); }
  __syncthreads();
  mx = s.maxkey; live = s.live;

  int token = -1, kept = 0;
  float logp = -INFINITY;
  if (live > 0u) {
    Place at;
    uint32_t nth = 0u;                        // the drawn token: the nth one (by index) of the value at.key
    at.key = mx; at.found = true;
    logp = 0.f; kept = 1;
    if (Tm > 0.f) {
      Row r;
      r.max = (double)value_of(mx); r.inv_t = 1.0 / (double)Tm;
      r.scale = (double)(1ull << (62 - (32 - __clz(V - 1 | 1))));
      uint32_t cm = 0u;
      unsigned long long mm = 0ull;
      for (int i = tid; i < V; i += THREADS) {
        const uint32_t key = key_of(load(l, i));
        if (!key) continue;
        const double e = real_weight(r, key);
        const unsigned long long w = __double2ull_rn(e * r.scale);
        add(s.top, key >> 21, w);
        if (e >= (double)min_p) { ++cm; mm += w; }
      }
      uint32_t cb, ct;
      unsigned long long mb, mt;
      __syncthreads();
      block_scan(s, cm, mm, cb, mb, ct, mt);
      const uint32_t n_min = ct;
      const unsigned long long mass_min = mt;
      uint32_t c2 = 0u;
      unsigned long long m2 = 0ull;
      for (int i = tid; i < BINS; i += THREADS) { c2 += s.top.count[i]; m2 += mass(s.top, i); }
      block_scan(s, c2, m2, cb, mb, ct, mt);
      uint32_t n = live;
      unsigned long long Wn = mt;
      if (k > 0 && (uint32_t)k < live) {
        const Place p = lookup(s, l, V, r, BY_RANK, (uint32_t)k - 1u, 0.0);
        n = (uint32_t)k;
        Wn = p.before_mass + (unsigned long long)(n - p.before_count) * weight(r, p.key);
      }
      if (top_p < 1.f) {
        const double x = (double)top_p * (double)Wn;
        const Place p = lookup(s, l, V, r, BY_MASS_BEFORE, 0u, x);
        uint32_t np = 1u;
        unsigned long long Wp = (unsigned long long)r.scale;
        if (x > 0.0 && p.found) {
          const unsigned long long w = weight(r, p.key);
          const double q = ceil((x - (double)p.before_mass) / (double)w);
          const uint32_t in = (uint32_t)fmin(fmax(q, 1.0), (double)p.count);
          np = p.before_count + in; Wp = p.before_mass + in * w;
        }
        if (np < n) { n = np; Wn = Wp; }
      }
      if (min_p > 0.f && n_min < n) {
        if (n_min > 0u) { n = n_min; Wn = mass_min; }
        else { n = 1u; Wn = (unsigned long long)r.scale; }
      }
      const float uf = a.u[row];
      const double u = uf > 0.f ? fmin((double)uf, 1.0 - 0x1p-24) : 0.0;
      const double x = u * (double)Wn;
      at = lookup(s, l, V, r, BY_MASS_UPTO, 0u, x);
      if (at.found) nth = (uint32_t)fmin(floor((x - (double)at.before_mass) / (double)weight(r, at.key)), (double)(at.count - 1u));
      if (!at.found || at.before_count + nth >= n) {               // rounding next to the last border: the last token that is kept
        at = lookup(s, l, V, r, BY_RANK, n - 1u, 0.0);
        nth = n - 1u - at.before_count;
      }
      logp = (float)(log_weight(r, at.key) - log((double)Wn / r.scale));
      kept = (int)n;
    }
    // the nth token of that value, by index
    uint32_t before = 0u;
    for (int i0 = 0; i0 < V; i0 += THREADS) {
      const int i = i0 + tid;
      const bool is = i < V && key_of(load(l, i)) == at.key;
      uint32_t cb, ct;
      unsigned long long mb, mt;
      block_scan(s, is ? 1u : 0u, 0ull, cb, mb, ct, mt);
      if (is && before + cb == nth) s.token = i;
      before += ct;
      if (before > nth) break;
    }
    __syncthreads();
    token = s.token;
  }
  if (tid == 0) {
    a.tokens[row] = token;
    if (a.next) a.next[row] = token;
    if (a.logprobs) a.logprobs[row] = logp;
    if (a.kept) a.kept[row] = kept;
  }
}

}  // namespace etxb_draw

extern "C" int32_t etxb_sample(int device, const etxb_sample_args* args, size_t bytes, void* cuda_stream) {
  using namespace etxb_draw;
  if (!args || bytes != sizeof(etxb_sample_args)) return etxb_host_fail(ETXB_E_ARG, "sample: needs an etxb_sample_args");
  if (device < 0 || device >= 64) return etxb_host_fail(ETXB_E_ARG, "sample: device index out of range");
  const etxb_sample_args a = *args;
  if (a.reserved != 0) return etxb_host_fail(ETXB_E_ARG, "sample: reserved is 0");
  if (a.rows < 0 || a.V < 1 || a.V > ETXB_SAMPLE_MAX_V) return etxb_host_fail(ETXB_E_UNSUPPORTED, "sample: rows >= 0 and 1 <= V <= 524288");
  if (a.dtype < ETXB_BF16 || a.dtype > ETXB_F32) return etxb_host_fail(ETXB_E_UNSUPPORTED, "sample: logits are bf16, fp16 or fp32");
  if (a.rows > 1 && a.row_stride < a.V) return etxb_host_fail(ETXB_E_ARG, "sample: rows overlap (row_stride < V)");
  if (a.rows == 0) return ETXB_OK;
  if (!a.logits || !a.u || !a.tokens) return etxb_host_fail(ETXB_E_ARG, "sample: logits, u and tokens are set");
  const uintptr_t size = a.dtype == ETXB_F32 ? 4 : 2;
  if (((uintptr_t)a.logits & (size - 1)) || (((uintptr_t)a.u | (uintptr_t)a.tokens | (uintptr_t)a.next | (uintptr_t)a.logprobs | (uintptr_t)a.kept | (uintptr_t)a.temperature |
      (uintptr_t)a.top_k | (uintptr_t)a.top_p | (uintptr_t)a.min_p) & 3)) return etxb_host_fail(ETXB_E_ARG, "sample: a pointer is not aligned to its elements");
  EtxbDeviceScope scope(device);
  ETXB_HOST_CU(scope.err);
  int sms = 0;
  ETXB_HOST_CU(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
  void* kargs[] = {(void*)&a};
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof cfg);
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  cfg.blockDim = dim3(THREADS); cfg.stream = (cudaStream_t)cuda_stream; cfg.attrs = &at; cfg.numAttrs = 1;
  // blocks of a row: as many as its counters need, and more while the device has room and each block still has 8192 logits
  int C = 1;
  const long long vectors = ((long long)a.V + 7 + 7) / 8;
  while ((vectors + C - 1) / C > CHUNK) C *= 2;
  const void* k;
  if (a.dtype == ETXB_F32 || C > MAX_CLUSTER) {
    k = a.dtype == ETXB_F32 ? (const void*)rows_kernel<float> : a.dtype == ETXB_F16 ? (const void*)rows_kernel<__half> : (const void*)rows_kernel<__nv_bfloat16>;
    C = 1;
    cfg.dynamicSmemBytes = sizeof(Shared);
  } else {
    while (C < MAX_CLUSTER && (long long)a.rows * 2 * C <= sms && vectors / C > 1024) C *= 2;
    const int nv = (int)((vectors + C - 1) / C + THREADS - 1) / THREADS;
    const bool half = a.dtype == ETXB_F16;
    k = nv <= 1 ? (half ? (const void*)counts_kernel<__half, 1> : (const void*)counts_kernel<__nv_bfloat16, 1>)
      : nv <= 2 ? (half ? (const void*)counts_kernel<__half, 2> : (const void*)counts_kernel<__nv_bfloat16, 2>)
      : nv <= 4 ? (half ? (const void*)counts_kernel<__half, 4> : (const void*)counts_kernel<__nv_bfloat16, 4>)
                : (half ? (const void*)counts_kernel<__half, 8> : (const void*)counts_kernel<__nv_bfloat16, 8>);
    cfg.dynamicSmemBytes = sizeof(Counts);
  }
  at.val.clusterDim.x = (unsigned)C; at.val.clusterDim.y = 1; at.val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)(a.rows * C));
  ETXB_HOST_CU(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)cfg.dynamicSmemBytes));
  ETXB_HOST_CU(cudaLaunchKernelExC(&cfg, k, kargs));
  return ETXB_OK;
}
