// Drawing tokens: temperature, top-k, top-p and min-p over rows of logits, with given random numbers (etxb_sample).
//
// Mathematics.  The live tokens of a row (neither -inf nor NaN) stand in the order "larger logit first, equal logits by index".  Token r of that order
// has the weight w_r = exp((l_r - l_0) / T).  Every cut keeps a beginning of the order:
//   top-k   the first min(k, live)                                          mass W_k = the sum of their weights
//   top-p   those with (sum of the weights before r) < p * W_k
//   min-p   those with w_r >= min_p
// so together they keep the first n (at least one).  Drawn is the first token whose inclusive sum exceeds u * W_n.
//
// The sums have to be right next to every border, and the order of atomics must not change them.  The bytes alone are 0.05 us for a row of 151936 and 12 us for 256;
// what bounds it is the way from one step of the definition to the next: blocks of a row that wait for each other, sums over all values, a place looked up in them.
//
// Logits of 16 bits (counts_kernel).  A row has at most 65536 different values, and a real one some thousands: the row is counted value by value, exactly, with
// 16-bit counters in shared memory, and then one exp in 64 bits per value that occurs, and sums over values in their order, give all three cuts and the
// draw.  Nothing is sorted.  A row belongs to a cluster of C blocks, each of which counts a part of it; values are joined through distributed shared
// memory, 32 neighbouring ones (a group) at a time, and only groups that occur.
//   32 rows of 151936 20 us (4 of them counting, at 0.2 clocks a logit; a lookup 1), one row 14, 256 rows 76 (1 TB/s), 8 rows of 4000 12.5.
// Logits of 32 bits (sums_kernel).  Bins by the first 11 bits of the value, then the next 11 and the last 10 of one bin: three passes for a border.  A bin has a
// number of tokens and a sum of weights, which are integers: exp in 64 bits times 2^S with S = 62 - ceil(log2 V), so that a row's sum fits 63 bits, is
// exact whatever the order, and a weight is off by 2^-(S+1) <= 2^-43 of the largest.
//   13 rows of 50257 36 us without cuts, 44 with top-k and top-p, 8 of them a lookup; 256 rows of 151936 467 and 473 (their bytes: 24), 64 rows 135: one block
//   a row (two for 64) keeps nothing of it on the chip and reads it again for every pass, and bins have more than LIST tokens.  Four copies
//   of the first bins, for four lanes each, gave nothing, nor did an exp in 32 bits (1 us): it is the passes and what the blocks wait for between them.
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
  if (a.next) a.next[row] = max(token, 0);                        // (a token there is: the next step looks it up)
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
// Keys: values as unsigned numbers in the values' order, two a word.  Numbers have the keys LOWEST .. HIGHEST; below them stand -inf (LOWEST - 1) and the
// NaN with a sign, above them the other NaN.  -0 has the key before +0's: counts of it become +0's.  INF: the bits of +inf (bf16 0x7f80, fp16 0x7c00).
constexpr uint32_t MINUS_ZERO = 0x7fffu, ZERO = 0x8000u;
template <uint32_t INF>
struct Key16 {
  static constexpr uint32_t LOWEST = 0x8000u - INF, HIGHEST = 0x8000u + INF, NOTHING = (0x8000u | INF) * 0x10001u;   // (two times -inf)
  static __device__ __forceinline__ uint32_t of_two(uint32_t u) {
    const uint32_t m = u & 0x80008000u;
    return u ^ 0x80008000u ^ (m - (m >> 15));
  }
  static __device__ __forceinline__ bool is(uint32_t k) { return k - LOWEST <= HIGHEST - LOWEST; }
};
template <typename T> __device__ __forceinline__ float value16(uint32_t key);
template <> __device__ __forceinline__ float value16<__nv_bfloat16>(uint32_t key) {
  return __uint_as_float(((key & 0x8000u) ? (key & 0x7fffu) : (~key & 0xffffu)) << 16);
}
template <> __device__ __forceinline__ float value16<__half>(uint32_t key) {
  return __half2float(__ushort_as_half((unsigned short)((key & 0x8000u) ? (key & 0x7fffu) : (~key & 0xffffu))));
}

constexpr int GROUPS = 2048, CHUNK = 8191;                          // groups of 32 values; vectors of 8 logits a block counts (16 bits hold their number)
constexpr int PIECE = 4095, PART = 32767, PARTS = 32;               // of a whole row (see counts_kernel)
struct Group {
  double mass, mass_min;                                            // sum of the weights of its tokens, and of those that min-p keeps
  uint32_t count, count_min;
};
struct Counts {
  uint32_t hist[32768];                                             // two counters a word
  Group group[GROUPS];                                              // of the whole row, those that occur, from the largest value down: each block joins a C-th of them
  double before_mass[GROUPS];                                       // and tells the others; of the groups before each
  uint32_t before_count[GROUPS];
  uint16_t list[GROUPS];                                            // which groups they are
  uint32_t bits[GROUPS / 32], row_bits[GROUPS / 32];                // the groups that occur in this block's part; in the row
  uint32_t part_key[PARTS], part_count[PARTS], n_parts, low;        // (a whole row) counts that 16 bits do not hold
  uint32_t maxkey;
  uint32_t at, nth, here;                                           // what was drawn: a value, and which of its tokens in this block
  int kept, mine;
  float logp;
  uint32_t entry, entry_before;
};
static_assert(sizeof(Counts) <= 231424, "a block's shared memory");

// NV > 0: a block has NV vectors a thread, which stay in registers.  NV = 0: one block counts a whole row, whatever its length, in pieces of PIECE vectors;
// before a counter could pass its 16 bits, what stands above 32767 in any of them goes to a list.
template <typename T, int NV>
__global__ void __launch_bounds__(THREADS, 1) counts_kernel(const etxb_sample_args a) {
  using K = Key16<sizeof(T) == 2 && __is_same(T, __half) ? 0x7c00u : 0x7f80u>;
  constexpr bool WHOLE = NV == 0;
  constexpr int N = WHOLE ? 4 : NV;
  extern __shared__ __align__(16) unsigned char smem[];
  Counts& s = *(Counts*)smem;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = WHOLE ? 1 : (int)cluster.num_blocks(), r = WHOLE ? 0 : (int)cluster.block_rank(), row = blockIdx.x / C;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = a.V;
  const Settings st = settings(a, row);
  const bool greedy = !(st.T > 0.f);

  // this block's vectors of 8 logits, from the last 16-byte boundary before the row on: logit v * 8 - shift + j
  const T* l = (const T*)a.logits + (long long)row * a.row_stride;
  const int shift = (int)((uintptr_t)l & 15) / 2, nvec = (shift + V + 7) / 8;
  const int v0 = (int)((long long)nvec * r / C), v1 = (int)((long long)nvec * (r + 1) / C);
  auto bits_of = [&](int v, int end) {                              // (-inf beside the row)
    uint4 q = make_uint4(K::NOTHING, K::NOTHING, K::NOTHING, K::NOTHING);
    const int e = v * 8 - shift;
    if (v < end && e >= 0 && e + 8 <= V) q = __ldg((const uint4*)(l + e));
    else if (v < end) {                                             // the row's ends, one by one
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int x = e + 2 * j;
        const uint32_t lo = x >= 0 && x < V ? ((const unsigned short*)l)[x] : K::NOTHING & 0xffffu, hi = x + 1 >= 0 && x + 1 < V ? ((const unsigned short*)l)[x + 1] : K::NOTHING & 0xffffu;
        w[j] = lo | (hi << 16);
      }
      q = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return q;
  };
  auto keys_of = [&](int v, int end) {
    const uint4 q = bits_of(v, end);
    return make_uint4(K::of_two(q.x), K::of_two(q.y), K::of_two(q.z), K::of_two(q.w));
  };
  uint4 key[N];
  uint32_t mx = 0u, low = 0u;
  auto fetch = [&](int v, int end) {
#pragma unroll
    for (int i = 0; i < N; ++i) key[i] = keys_of(v + i * THREADS + tid, end);
  };
  auto largest = [&]() {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t k = ((const uint32_t*)&key[i])[j >> 1] >> (16 * (j & 1)) & 0xffffu;
        if (K::is(k)) mx = max(mx, k == MINUS_ZERO ? ZERO : k);
      }
  };
  // No branch for a logit (with one for "-inf" and one for the lowest number 0.46 clocks each, so 0.2; the atomics alone, into 65536 counters, 0.14).  Masked ones, -inf or the type's lowest
  // number, are most of some rows and would wait for each other: the first are not counted, the others without memory.
  const uint32_t hist = (uint32_t)__cvta_generic_to_shared(s.hist);
  auto count = [&]() {
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t w = ((const uint32_t*)&key[i])[j >> 1], k = j & 1 ? w >> 16 : w & 0xffffu;
        asm volatile("{\n .reg .pred p;\n setp.gt.u32 p, %1, 1;\n @p red.shared.add.u32 [%2], %3;\n @!p add.u32 %0, %0, %1;\n}" : "+r"(low) :
                         "r"(k - (K::LOWEST - 1u)), "r"(hist + ((k << 1) & 0x1fffcu)), "r"(k & 1u ? 0x10000u : 1u) : "memory");
      }
    }
  };
  if constexpr (!WHOLE) fetch(v0, v1);
  if (!greedy) {
    for (int i = tid; i < 32768 / 4; i += THREADS) ((uint4*)s.hist)[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  if (tid == 0) { s.maxkey = 0u; s.n_parts = 0u; s.low = 0u; }
  __syncthreads();
  if constexpr (!WHOLE) {
    if (greedy) largest(); else count();
  } else {
    for (int v = 0, piece = 0; v < nvec; v += PIECE, ++piece) {
      fetch(v, min(v + PIECE, nvec));
      if (greedy) { largest(); continue; }
      if (piece >= 2) {                                             // two pieces are 65520 logits; behind this, 32768 and one piece fit
        __syncthreads();
        for (int i = tid; i < 32768 / 4; i += THREADS) {
          const uint4 q = ((const uint4*)s.hist)[i];
          if (((q.x | q.y | q.z | q.w) & 0x80008000u) == 0u) continue;
          for (int k = 8 * i; k < 8 * i + 8; ++k) {
            uint16_t& c = ((uint16_t*)s.hist)[k];
            if (c < PART + 1) continue;
            c -= PART;
            if (K::is((uint32_t)k)) { const uint32_t n = atomicAdd(&s.n_parts, 1u); s.part_key[n] = k == MINUS_ZERO ? ZERO : k; s.part_count[n] = PART; }      // (16 of them at most)
          }
        }
        __syncthreads();
      }
      count();
    }
  }
  if (greedy) {
    mx = __reduce_max_sync(~0u, mx);
    if (lane == 0) atomicMax(&s.maxkey, mx);
    __syncthreads();
  } else {
    low = __reduce_add_sync(~0u, low);
    if (lane == 0 && low) atomicAdd(&s.low, low);
    __syncthreads();
    // what is no number goes, -0 becomes +0, the lowest ones come in
    if (tid < (int)K::LOWEST / 2) s.hist[tid] = 0u;
    if (tid < (0x10000 - (int)K::HIGHEST) / 2) s.hist[K::HIGHEST / 2 + tid] &= tid ? 0u : 0xffffu;
    static_assert(K::LOWEST / 2 <= THREADS && (0x10000 - K::HIGHEST) / 2 <= THREADS && K::HIGHEST % 2 == 0 && K::LOWEST % 2 == 0, "a thread a word");
    if (tid == THREADS - 1) {
      auto put = [&](uint32_t k, uint32_t n) {
        uint16_t& c = ((uint16_t*)s.hist)[k];
        if (c + n > 65535u) { const uint32_t i = s.n_parts++; s.part_key[i] = k; s.part_count[i] = n - 1u; n = 1u; if (c) { s.part_count[i] += 1u; n = 0u; } }
        c += (uint16_t)n;
      };
      const uint32_t minus = s.hist[MINUS_ZERO / 2] >> 16;
      if (minus) { s.hist[MINUS_ZERO / 2] &= 0xffffu; put(ZERO, minus); }
      if (s.low) put(K::LOWEST, s.low);
    }
    __syncthreads();
    // groups that occur: four lanes look at the 64 bytes of one; the largest value
    for (int i = 0; i < GROUPS * 4 / THREADS; ++i) {
      const uint4 q = ((const uint4*)s.hist)[i * THREADS + tid];
      uint32_t any = q.x | q.y | q.z | q.w;
      if (any) {
        const int top = q.w ? 6 : q.z ? 4 : q.y ? 2 : 0;
        mx = (uint32_t)((i * THREADS + tid) * 8 + top) + ((q.w ? q.w : q.z ? q.z : q.y ? q.y : q.x) >> 16 ? 1u : 0u);         // (i rises)
      }
      any |= __shfl_xor_sync(~0u, any, 1); any |= __shfl_xor_sync(~0u, any, 2);
      uint32_t b = __ballot_sync(~0u, any != 0u);                   // 8 groups, a nibble each
      if (lane == 0) {
        b &= 0x11111111u;
        b = (b | b >> 3) & 0x03030303u; b = (b | b >> 6) & 0x000f000fu; b = (b | b >> 12) & 0xffu;
        ((unsigned char*)s.bits)[i * (THREADS / 32) + warp] = (unsigned char)b;
      }
    }
    mx = __reduce_max_sync(~0u, mx);
    if (lane == 0) atomicMax(&s.maxkey, mx);
  }
  cluster.sync();
  // one word from every block of the cluster, all on their way at once
  auto from_all = [&](const void* mine, auto type, auto use) {
    decltype(type) v[MAX_CLUSTER];
#pragma unroll
    for (int c = 0; c < MAX_CLUSTER; ++c) if (c < C) v[c] = *(const decltype(type)*)cluster.map_shared_rank((void*)mine, c);
#pragma unroll
    for (int c = 0; c < MAX_CLUSTER; ++c) if (c < C) use(c, v[c]);
  };
  uint32_t maxkey = 0u;
  int first_with_max = 0;
  from_all(&s.maxkey, uint32_t(), [&](int c, uint32_t m) { if (m > maxkey) { maxkey = m; first_with_max = c; } });
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
    for (uint32_t i = 0; i < s.n_parts; ++i) n += s.part_key[i] == k ? s.part_count[i] : 0u;      // (of this block: it is the only one, or there are none)
    from_all((const uint16_t*)s.hist + k, uint16_t(), [&](int, uint16_t x) { n += x; });
    return n;
  };

  if (greedy) {
    if (tid == 0) { s.at = maxkey; s.nth = 0u; s.kept = 1; s.logp = 0.f; s.mine = r == first_with_max; }
  } else {
    // the row's groups that occur, in descending order
    if (tid < GROUPS / 32) {
      uint32_t b = 0u;
      from_all(&s.bits[tid], uint32_t(), [&](int, uint32_t x) { b |= x; });
      s.row_bits[tid] = b;
    }
    __syncthreads();
    static_assert(GROUPS == 2 * THREADS, "two words of 32 groups a warp");
    const uint32_t bits0 = s.row_bits[warp], bits1 = s.row_bits[WARPS + warp], c0 = (uint32_t)__popc(s.row_bits[lane]), c1 = (uint32_t)__popc(s.row_bits[WARPS + lane]);
    const uint32_t upper = __reduce_add_sync(~0u, c1), groups = upper + __reduce_add_sync(~0u, c0), above = ~((2u << lane) - 1u);
    const uint32_t first1 = __reduce_add_sync(~0u, lane > warp ? c1 : 0u), first0 = upper + __reduce_add_sync(~0u, lane > warp ? c0 : 0u);
    if (bits1 >> lane & 1u) s.list[first1 + (uint32_t)__popc(bits1 & above)] = (uint16_t)(THREADS + tid);
    if (bits0 >> lane & 1u) s.list[first0 + (uint32_t)__popc(bits0 & above)] = (uint16_t)tid;
    __syncthreads();
    // each block joins every C-th, a warp a group
    for (uint32_t i = (uint32_t)(r + C * warp); i < groups; i += (uint32_t)(C * WARPS)) {
      const uint32_t k = s.list[i] * 32u + 31u - (uint32_t)lane;                                   // lanes from the group's largest value down
      const uint32_t n = tokens_of(k);
      const double w = n ? weight(k) : 0.0;
      const bool in = n && w >= (double)st.min_p;
      double m = (double)n * w, mm = in ? m : 0.0;
#pragma unroll
      for (int o = 16; o; o >>= 1) { m += __shfl_xor_sync(~0u, m, o); mm += __shfl_xor_sync(~0u, mm, o); }
      Group x;
      x.mass = m; x.mass_min = mm; x.count = __reduce_add_sync(~0u, n); x.count_min = __reduce_add_sync(~0u, in ? n : 0u);
      if (lane < C) *cluster.map_shared_rank(&s.group[i], lane) = x;
    }
    cluster.sync();
    if (warp == 0) {
      // tokens and mass before each group: a lane has a 32nd of them (a real row has some hundred groups; all warps and two barriers took 1.5 us)
      const uint32_t per = (groups + 31u) / 32u, i0 = min(lane * per, groups), i1 = min(i0 + per, groups);
      uint32_t own_c = 0u, total_min = 0u;
      double own_m = 0.0, total_mm = 0.0;
      for (uint32_t i = i0; i < i1; ++i) { const Group x = s.group[i]; own_c += x.count; own_m += x.mass; total_min += x.count_min; total_mm += x.mass_min; }
      uint32_t cb = own_c;
      double mb = own_m;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(~0u, cb, o);
        const double z = __shfl_up_sync(~0u, mb, o);
        if (lane >= o) { cb += y; mb += z; }
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) total_mm += __shfl_xor_sync(~0u, total_mm, o);
      total_min = __reduce_add_sync(~0u, total_min);
      const uint32_t total = __shfl_sync(~0u, cb, 31);
      const double total_m = __shfl_sync(~0u, mb, 31), up_m = __shfl_up_sync(~0u, mb, 1);
      cb -= own_c; mb = lane ? up_m : 0.0;
      for (uint32_t i = i0; i < i1; ++i) { s.before_count[i] = cb; s.before_mass[i] = mb; cb += s.group[i].count; mb += s.group[i].mass; }
      __syncwarp();
      // A border: the group it falls into -- the last that begins at or before it, found 32 at a time -- and then the value in it, a lane each.
      uint32_t place_key = 0u, place_before = 0u, place_count = 0u;
      double place_mass = 0.0, place_weight = 1.0;
      auto lookup = [&](int how, uint32_t rank, double y) {
        auto begins = [&](uint32_t i) { return how == BY_RANK ? s.before_count[i] <= rank : how == BY_MASS_BEFORE ? s.before_mass[i] < y : s.before_mass[i] <= y; };
        // (beginnings do not fall, but by a rounding between two groups that hold next to nothing: the last one that holds is taken)
        uint32_t i = per * (31u - (uint32_t)__clz(__ballot_sync(~0u, lane * per < groups && begins(lane * per)) | 1u));
        const uint32_t low = __ballot_sync(~0u, (uint32_t)lane < per && i + lane < groups && begins(i + lane)) | 1u;
        const uint32_t high = __ballot_sync(~0u, 32u + lane < per && i + 32u + lane < groups && begins(i + 32u + lane));
        i += high ? 63u - (uint32_t)__clz(high) : 31u - (uint32_t)__clz(low);
        const uint32_t k = s.list[i] * 32u + 31u - (uint32_t)lane, n = tokens_of(k);
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
        cb += s.before_count[i];
        const double m0 = s.before_mass[i] + mbef, m1 = s.before_mass[i] + m;
        uint32_t hits = __ballot_sync(~0u, n && falls(how, rank, y, cb, n, m0, m1));
        // (sums within a group are rounded apart from the group's: a border on its very end belongs to its last value)
        if (!hits) hits = 1u << (31 - __clz(__ballot_sync(~0u, n != 0u)));
        const int x1 = __ffs(hits) - 1;
        place_key = __shfl_sync(~0u, k, x1); place_before = __shfl_sync(~0u, cb, x1); place_count = __shfl_sync(~0u, n, x1);
        place_mass = __shfl_sync(~0u, m0, x1); place_weight = __shfl_sync(~0u, w, x1);
      };
      uint32_t n = total;
      double Wn = total_m;
      if (st.k > 0 && (uint32_t)st.k < total) {
        lookup(BY_RANK, (uint32_t)st.k - 1u, 0.0);
        n = (uint32_t)st.k;
        Wn = place_mass + (double)(n - place_before) * place_weight;
      }
      if (st.top_p < 1.f) {
        const double y = (double)st.top_p * Wn;
        uint32_t np = 1u;
        double Wp = 1.0;
        if (y > 0.0) {
          lookup(BY_MASS_BEFORE, 0u, y);
          const double q = ceil((y - place_mass) / place_weight);
          const uint32_t in = (uint32_t)fmin(fmax(q, 1.0), (double)place_count);
          np = place_before + in; Wp = place_mass + (double)in * place_weight;
        }
        if (np < n) { n = np; Wn = Wp; }
      }
      if (st.min_p > 0.f && total_min < n) {
        n = total_min ? total_min : 1u;
        Wn = total_min ? total_mm : 1.0;
      }
      const double y = st.u * Wn;
      lookup(BY_MASS_UPTO, 0u, y);
      uint32_t nth = (uint32_t)fmin(fmax(floor((y - place_mass) / place_weight), 0.0), (double)(place_count - 1u));
      if (place_before + nth >= n) {                                // rounding next to the last border: the last token that is kept
        lookup(BY_RANK, n - 1u, 0.0);
        nth = n - 1u - place_before;
      }
      // which block has it: the tokens of that value in the blocks before
      uint32_t ahead = 0u, here = 0u;
      if constexpr (WHOLE) here = place_count;
      else from_all((const uint16_t*)s.hist + place_key, uint16_t(), [&](int c, uint16_t z) { if (c < r) ahead += z; if (c == r) here = z; });
      if (lane == 0) {
        s.at = place_key; s.nth = nth - ahead; s.mine = ahead <= nth && nth < ahead + here;
        s.kept = (int)n; s.logp = (float)(log_weight(place_key) - log(Wn));
      }
    }
  }
  __syncthreads();
  // nobody reads another block's memory from here on; a block leaves when all have come so far
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  const uint32_t at = s.at, nth = s.nth;
  const float logp = s.logp;
  const int kept = s.kept;
  const bool mine = s.mine != 0;
  const uint32_t at_too = at == ZERO ? MINUS_ZERO : at;
  // Most vectors have none: both halves of four words are looked at together, where a borrow from a lower half that is equal may take the upper one along.
  auto some = [&](const uint4& q, uint32_t care, uint32_t is) {
    uint32_t m = 0u;
#pragma unroll
    for (int j = 0; j < 4; ++j) { const uint32_t x = ((&q.x)[j] & care) ^ is; m |= (x - 0x00010001u) & ~x; }
    return (m & 0x80008000u) != 0u;
  };
  auto matches = [&](const uint4& q) {
    uint32_t m = 0u;
#pragma unroll
    for (int j = 0; j < 8; ++j) { const uint32_t k = (&q.x)[j >> 1] >> (16 * (j & 1)) & 0xffffu; m |= (k == at || k == at_too ? 1u : 0u) << j; }
    return m;
  };
  if constexpr (WHOLE) {
    // a warp has a 32nd of the row, in the order of the indices
    uint32_t* cnt = (uint32_t*)s.list;
    const int per = (nvec + WARPS - 1) / WARPS, w0 = min(warp * per, nvec), w1 = min(w0 + per, nvec);
    const uint32_t care = at == ZERO ? 0x7fff7fffu : ~0u, is = (at & 0x8000u ? at & 0x7fffu : ~at & 0xffffu) * 0x10001u;
    uint32_t c = 0u;
#pragma unroll 4
    for (int v = w0; v < w1; v += 32) {
      const uint4 q = bits_of(v + lane, w1);
      if (some(q, care, is)) c += (uint32_t)__popc(matches(make_uint4(K::of_two(q.x), K::of_two(q.y), K::of_two(q.z), K::of_two(q.w))));
    }
    c = __reduce_add_sync(~0u, c);
    if (lane == 0) cnt[warp] = c;
    __syncthreads();
    uint32_t before = 0u;
    for (int w = 0; w < warp; ++w) before += cnt[w];
    if (before <= nth && nth < before + c)
      for (int v = w0; v < w1; v += 32) {
        uint32_t m = matches(keys_of(v + lane, w1));
        const uint32_t n = (uint32_t)__popc(m);
        if (!__any_sync(~0u, m != 0u)) continue;
        uint32_t upto = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const uint32_t x = __shfl_up_sync(~0u, upto, o); if (lane >= o) upto += x; }
        const uint32_t mine_before = before + upto - n;
        if (mine_before <= nth && nth < mine_before + n) {
          for (uint32_t q = mine_before; q < nth; ++q) m &= m - 1u;
          store(a, row, (v + lane) * 8 - shift + __ffs(m) - 1, logp, kept);
        }
        before += __shfl_sync(~0u, upto, 31);
        if (before > nth) break;
      }
  } else if (mine) {
    uint32_t* cnt = (uint32_t*)s.list;                              // matches by vector number and warp: the order of the indices
    uint32_t match[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      match[i] = at == ZERO || some(key[i], ~0u, at * 0x10001u) ? matches(key[i]) : 0u;
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
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ================================================================================================ logits of 32 bits
// Logits as keys whose order as unsigned numbers is the order of the values; 0: not live (-inf, NaN).  -0 counts as +0.
__device__ __forceinline__ uint32_t key_of(float l) {
  uint32_t u = __float_as_uint(l);
  if ((u << 1) > 0xff000000u || u == 0xff800000u) return 0u;
  if ((u << 1) == 0u) u = 0u;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key); }

constexpr int BINS = 2048, LIST = 2048;
struct Sums {
  uint32_t count[BINS], lo[BINS], hi[BINS];                         // of this block's part
  uint32_t all_count[2][BINS];                                      // of the row: by the first 11 bits of the key; by the next ones of one of those bins
  unsigned long long all_mass[2][BINS];
  uint32_t wc[WARPS], wcm[WARPS];
  unsigned long long wm[WARPS], wmm[WARPS];
  uint32_t maxkey, live, kept_min, here;
  unsigned long long mass_min;
  uint32_t bin, before_count, n, found;
  unsigned long long before_mass;
  uint32_t part[2][LIST], n_part[2], list[LIST];                    // the values of one of the first bins: this block's, and the row's
};
struct Row {
  double max, inv_t;
  double scale;                               // 2^S
};
__device__ __forceinline__ double log_weight(const Row& r, uint32_t key) {
  const double d = (double)value_of(key) - r.max;
  return d == d ? d * r.inv_t : 0.0;          // (inf - inf: the largest itself)
}
__device__ __noinline__ double exponential(double x) { return exp(x); }   // (one place in the code: three inlined were slower by a twentieth)
__device__ __forceinline__ double real_weight(const Row& r, uint32_t key) {
  const double d = (double)value_of(key) - r.max;
  return d < 0.0 ? (d == -INFINITY ? 0.0 : exponential(d * r.inv_t)) : 1.0;     // (beside an infinite logit a finite one has none, at any temperature)
}
__device__ __forceinline__ unsigned long long weight(const Row& r, uint32_t key) { return __double2ull_rn(real_weight(r, key) * r.scale); }

// C blocks have a row together.  Each goes over its part of it twice for the first bins.  A border falls into one of them, which rarely has more than LIST tokens: they are
// told to all blocks, and each refines them by itself.  (Refined over the row, with the blocks' bins joined for each level: 13 rows of 50257 67 us.)  A bin of more tokens
// is refined over the row.
__global__ void __launch_bounds__(THREADS) sums_kernel(const etxb_sample_args a) {
  extern __shared__ __align__(16) unsigned char smem[];
  Sums& s = *(Sums*)smem;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), r = (int)cluster.block_rank(), row = blockIdx.x / C;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int i0 = (int)((long long)a.V * r / C), i1 = (int)((long long)a.V * (r + 1) / C);
  const float* l = (const float*)a.logits + (long long)row * a.row_stride;
  const Settings st = settings(a, row);

  if (tid == 0) { s.maxkey = 0u; s.live = 0u; s.kept_min = 0u; s.mass_min = 0ull; }
  auto clear = [&]() { for (int i = tid; i < BINS; i += THREADS) { s.count[i] = 0u; s.lo[i] = 0u; s.hi[i] = 0u; } };
  clear();
  __syncthreads();
  uint32_t mx = 0u, live = 0u;
  // four loads ahead
  auto for_all = [&](auto use) {
    auto at = [&](int i) { return i < i1 ? l[i] : -INFINITY; };
    float x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = at(i0 + tid + j * THREADS);
#pragma unroll 1
    for (int i = i0 + tid; i < i1; i += 4 * THREADS)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t k = key_of(x[j]);
        x[j] = at(i + (4 + j) * THREADS);
        use(k);
      }
  };
  for_all([&](uint32_t key) { mx = max(mx, key); live += key ? 1u : 0u; });
  mx = __reduce_max_sync(~0u, mx); live = __reduce_add_sync(~0u, live);
  if (lane == 0) { atomicMax(&s.maxkey, mx); atomicAdd(&s.live, live); }
  cluster.sync();
  mx = live = 0u;
  for (int c = 0; c < C; ++c) { mx = max(mx, *cluster.map_shared_rank(&s.maxkey, c)); live += *cluster.map_shared_rank(&s.live, c); }

  int token = -1, kept = 0;
  float logp = -INFINITY;
  uint32_t at = mx, nth = 0u;                 // the drawn token: the nth one (by index) of that value
  if (live > 0u) { logp = 0.f; kept = 1; }
  if (live > 0u && st.T > 0.f) {
    Row w;
    w.max = (double)value_of(mx); w.inv_t = 1.0 / (double)st.T;
    w.scale = (double)(1ull << (62 - (32 - __clz((a.V - 1) | 1))));
    auto add = [&](uint32_t i, unsigned long long x) {
      atomicAdd(&s.count[i], 1u);
      const uint32_t lo = (uint32_t)x;
      uint32_t hi = (uint32_t)(x >> 32);
      if (lo) { const uint32_t old = atomicAdd(&s.lo[i], lo); hi += (old + lo < old) ? 1u : 0u; }
      if (hi) atomicAdd(&s.hi[i], hi);
    };
    // the blocks' bins into the row's, which every block gets
    auto join = [&](int level) {
      cluster.sync();
      for (int i = r * (BINS / C) + tid; i < (r + 1) * (BINS / C); i += THREADS) {
        uint32_t n = 0u;
        unsigned long long m = 0ull;
#pragma unroll
        for (int c = 0; c < MAX_CLUSTER; ++c)
          if (c < C) {
            const Sums* o = cluster.map_shared_rank(&s, c);
            n += o->count[i]; m += ((unsigned long long)o->hi[i] << 32) + o->lo[i];
          }
        for (int c = 0; c < C; ++c) { Sums* o = cluster.map_shared_rank(&s, c); o->all_count[level][i] = n; o->all_mass[level][i] = m; }
      }
      cluster.sync();
    };
    uint32_t cm = 0u;
    unsigned long long mm = 0ull;
    for_all([&](uint32_t key) {
      if (!key) return;
      const double e = real_weight(w, key);
      const unsigned long long x = __double2ull_rn(e * w.scale);
      add(key >> 21, x);
      if (e >= (double)st.min_p) { ++cm; mm += x; }
    });
    cm = __reduce_add_sync(~0u, cm);
#pragma unroll
    for (int o = 16; o; o >>= 1) mm += __shfl_xor_sync(~0u, mm, o);
    if (lane == 0) { atomicAdd(&s.kept_min, cm); atomicAdd(&s.mass_min, mm); }
    join(0);
    uint32_t n_min = 0u;
    unsigned long long mass_min = 0ull;
    for (int c = 0; c < C; ++c) { n_min += *cluster.map_shared_rank(&s.kept_min, c); mass_min += *cluster.map_shared_rank(&s.mass_min, c); }
    // A thread's two bins (in descending order), with the tokens and the mass of those before them.
    struct Two { uint32_t c[2], before; unsigned long long m[2], mass; };
    unsigned long long total = 0ull;
    auto scan = [&](int level, int nbins) {
      Two b;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int i = nbins - 1 - (2 * tid + k);
        b.c[k] = i >= 0 ? s.all_count[level][i] : 0u; b.m[k] = i >= 0 ? s.all_mass[level][i] : 0ull;
      }
      uint32_t ci = b.c[0] + b.c[1];
      unsigned long long mi = b.m[0] + b.m[1];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(~0u, ci, o);
        const unsigned long long z = __shfl_up_sync(~0u, mi, o);
        if (lane >= o) { ci += y; mi += z; }
      }
      __syncthreads();
      if (lane == 31) { s.wc[warp] = ci; s.wm[warp] = mi; }
      __syncthreads();
      uint32_t cw = s.wc[lane];
      unsigned long long mw = s.wm[lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(~0u, cw, o);
        const unsigned long long z = __shfl_up_sync(~0u, mw, o);
        if (lane >= o) { cw += y; mw += z; }
      }
      total = __shfl_sync(~0u, mw, 31);
      const uint32_t cb = __shfl_sync(~0u, cw, (warp + 31) & 31);
      const unsigned long long mb = __shfl_sync(~0u, mw, (warp + 31) & 31);
      b.before = (warp ? cb : 0u) + ci - b.c[0] - b.c[1]; b.mass = (warp ? mb : 0ull) + mi - b.m[0] - b.m[1];
      return b;
    };
    // the bin that a lookup falls into, given the tokens and mass before all of them: s.bin, or ~0
    auto pick = [&](const Two& b, int nbins, int how, uint32_t rank, double x, uint32_t c0, unsigned long long m0) {
      __syncthreads();                        // (the last lookup's bin is read)
      if (tid == 0) s.bin = ~0u;
      __syncthreads();
      uint32_t ci = c0 + b.before;
      unsigned long long mi = m0 + b.mass;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (falls(how, rank, x, ci, b.c[k], mi, mi + b.m[k])) { s.bin = (uint32_t)(nbins - 1 - (2 * tid + k)); s.before_count = ci; s.before_mass = mi; s.n = b.c[k]; }
        ci += b.c[k]; mi += b.m[k];
      }
      __syncthreads();
    };
    const Two first = scan(0, BINS);          // (the same for every lookup)
    uint32_t place_key = 0u, place_before = 0u, place_count = 0u;
    unsigned long long place_mass = 0ull;
    uint32_t held = ~0u;                      // the bin whose tokens s.list has
    int buf = 0;
    auto lookup = [&](int how, uint32_t rank, double x) {
      pick(first, BINS, how, rank, x, 0u, 0ull);
      if (s.bin == ~0u) return false;
      uint32_t prefix = s.bin, cb = s.before_count;
      unsigned long long mb = s.before_mass;
      const uint32_t in_bin = s.n;
      const bool few = in_bin <= LIST;        // (of the whole row: every block decides alike)
      if (few && prefix != held) {
        if (tid == 0) s.n_part[buf] = 0u;
        __syncthreads();
        for_all([&](uint32_t k) { if (k && k >> 21 == prefix) s.part[buf][atomicAdd(&s.n_part[buf], 1u)] = k; });
        cluster.sync();                       // (a block reads another one's part until the next such sync: the parts alternate)
        uint32_t off = 0u, n[MAX_CLUSTER];
#pragma unroll
        for (int c = 0; c < MAX_CLUSTER; ++c) n[c] = c < C ? *cluster.map_shared_rank(&s.n_part[buf], c) : 0u;
#pragma unroll
        for (int c = 0; c < MAX_CLUSTER; ++c) {
          if (c >= C) break;
          const uint32_t* from = cluster.map_shared_rank(s.part[buf], c);
          for (uint32_t i = tid; i < n[c]; i += THREADS) s.list[off + i] = from[i];
          off += n[c];
        }
        held = prefix; buf ^= 1;
        __syncthreads();
      }
      for (int level = 1; level < 3; ++level) {
        const int bits = level == 1 ? 11 : 10, shift = level == 1 ? 10 : 0, nb = 1 << bits;
        clear();
        __syncthreads();
        auto take = [&](uint32_t k) { if (k && (k >> (shift + bits)) == prefix) add((k >> shift) & (nb - 1), weight(w, k)); };
        if (few) {
          for (uint32_t i = tid; i < in_bin; i += THREADS) take(s.list[i]);
          __syncthreads();
          for (int i = tid; i < BINS; i += THREADS) { s.all_count[1][i] = s.count[i]; s.all_mass[1][i] = ((unsigned long long)s.hi[i] << 32) + s.lo[i]; }
          __syncthreads();
        } else {
          for_all(take);
          join(1);
        }
        pick(scan(1, nb), nb, how, rank, x, cb, mb);
        if (s.bin == ~0u) return false;       // (cannot be: the sums of a bin are the bin's)
        prefix = (prefix << bits) | s.bin; cb = s.before_count; mb = s.before_mass;
        if (few && level == 1 && s.n == 1u) { // one token: its value needs no more bins
          for (uint32_t i = tid; i < in_bin; i += THREADS) if (s.list[i] >> 10 == prefix) s.found = s.list[i];
          __syncthreads();
          prefix = s.found;
          break;
        }
      }
      place_key = prefix; place_before = cb; place_mass = mb; place_count = s.n;
      return true;
    };
    uint32_t n = live;
    unsigned long long Wn = total;            // (of the first bins: the last scan is theirs)
    // top-k, top-p, the draw, and the last token that is kept where rounding next to the last border asks for it
#pragma unroll 1
    for (int stage = 0; stage < 4; ++stage) {
      int how = BY_RANK;
      uint32_t rank = 0u;
      double x = 0.0;
      if (stage == 0) {
        if (!(st.k > 0 && (uint32_t)st.k < live)) continue;
        rank = (uint32_t)st.k - 1u;
      } else if (stage == 1) {
        if (!(st.top_p < 1.f)) continue;
        how = BY_MASS_BEFORE; x = (double)st.top_p * (double)Wn;
        if (!(x > 0.0)) { n = 1u; Wn = (unsigned long long)w.scale; continue; }
      } else if (stage == 2) {
        if (st.min_p > 0.f && n_min < n) {
          n = n_min ? n_min : 1u;
          Wn = n_min ? mass_min : (unsigned long long)w.scale;
        }
        how = BY_MASS_UPTO; x = st.u * (double)Wn;
      } else {
        if (place_before + nth < n) break;
        rank = n - 1u;
      }
      const bool found = lookup(how, rank, x);
      const unsigned long long y = weight(w, place_key);
      if (stage == 0) {
        n = (uint32_t)st.k;
        Wn = place_mass + (unsigned long long)(n - place_before) * y;
      } else if (stage == 1) {
        uint32_t np = 1u;
        unsigned long long Wp = (unsigned long long)w.scale;
        if (found) {
          const uint32_t in = (uint32_t)fmin(fmax(ceil((x - (double)place_mass) / (double)y), 1.0), (double)place_count);
          np = place_before + in; Wp = place_mass + in * y;
        }
        if (np < n) { n = np; Wn = Wp; }
      } else if (stage == 2) {
        if (found) nth = (uint32_t)fmin(fmax(floor((x - (double)place_mass) / (double)y), 0.0), (double)(place_count - 1u));
        else { place_before = n; nth = 0u; }                        // (rounding next to the last border)
      } else nth = n - 1u - place_before;
    }
    at = place_key;
    logp = (float)(log_weight(w, at) - log((double)Wn / w.scale));
    kept = (int)n;
  }
  if (live == 0u) {
    if (r == 0 && tid == 0) store(a, row, token, logp, kept);
    cluster.sync();
    return;
  }
  // its nth token, by index: a warp has 32nd parts of the block's part
  const int per = (i1 - i0 + WARPS - 1) / WARPS, w0 = i0 + warp * per, w1 = min(i1, w0 + per);
  uint32_t c = 0u;
#pragma unroll 4
  for (int i = w0 + lane; i < w1; i += 32) c += key_of(l[i]) == at ? 1u : 0u;
  c = __reduce_add_sync(~0u, c);
  if (tid == 0) s.here = 0u;
  __syncthreads();
  if (lane == 0) { s.wcm[warp] = c; atomicAdd(&s.here, c); }
  cluster.sync();
  uint32_t before = 0u;
  for (int b = 0; b < r; ++b) before += *cluster.map_shared_rank(&s.here, b);
  for (int b = 0; b < warp; ++b) before += s.wcm[b];
  if (before <= nth && nth < before + c)
    for (int i = w0; i < w1; i += 32) {
      const bool is = i + lane < w1 && key_of(l[i + lane]) == at;
      uint32_t hits = __ballot_sync(~0u, is);
      const uint32_t some = (uint32_t)__popc(hits);
      if (nth < before + some) {
        for (uint32_t q = before; q < nth; ++q) hits &= hits - 1u;
        if (lane == 0) store(a, row, i + __ffs(hits) - 1, logp, kept);
        break;
      }
      before += some;
    }
  cluster.sync();                                                   // (no block leaves while another one reads its memory)
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
  ETXB_HOST_CU(etxb_host_sms(device, &sms));
  void* kargs[] = {(void*)&a};
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof cfg);
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  cfg.blockDim = dim3(THREADS); cfg.stream = (cudaStream_t)cuda_stream; cfg.attrs = &at; cfg.numAttrs = 1;
  int C = 1;
  static std::atomic<char> ready[11][64];
  const void* k;
  int which;
  if (a.dtype == ETXB_F32) {
    k = (const void*)sums_kernel; which = 10;
    while (C < MAX_CLUSTER && (long long)a.rows * 2 * C <= sms && a.V / C > 2048) C *= 2;
    cfg.dynamicSmemBytes = sizeof(Sums);
  } else {
    static const void* const kernels[2][5] = {
        {(const void*)counts_kernel<__nv_bfloat16, 0>, (const void*)counts_kernel<__nv_bfloat16, 1>, (const void*)counts_kernel<__nv_bfloat16, 2>, (const void*)counts_kernel<__nv_bfloat16, 4>,
         (const void*)counts_kernel<__nv_bfloat16, 8>},
        {(const void*)counts_kernel<__half, 0>, (const void*)counts_kernel<__half, 1>, (const void*)counts_kernel<__half, 2>, (const void*)counts_kernel<__half, 4>, (const void*)counts_kernel<__half, 8>}};
    // Blocks of a row: as many as its counters need, and more while the device has room and each block still has 8192 logits.  Where more than twice the device's blocks
    // would come of it, or too many for a cluster, one block has a whole row (rows of 151936, us: 64 in four blocks each 40, the largest of them 21; 100 in one each 41, 25,
    // where four each would take three rounds of the 21 that 32 rows take; 256 in one each 78).
    const long long vectors = ((long long)a.V + 7 + 7) / 8;
    int size = 0;
    while ((vectors + C - 1) / C > CHUNK) C *= 2;
    if (C > MAX_CLUSTER || (C > 1 && (long long)a.rows * C > 2 * sms)) C = 1;
    else {
      while (C < MAX_CLUSTER && (long long)a.rows * 2 * C <= sms && vectors / C > 1024) C *= 2;
      const int nv = ((int)((vectors + C - 1) / C) + THREADS - 1) / THREADS;
      size = nv <= 1 ? 1 : nv <= 2 ? 2 : nv <= 4 ? 3 : 4;
    }
    k = kernels[a.dtype == ETXB_F16][size]; which = 5 * (a.dtype == ETXB_F16) + size;
    cfg.dynamicSmemBytes = sizeof(Counts);
  }
  at.val.clusterDim.x = (unsigned)C; at.val.clusterDim.y = 1; at.val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)(a.rows * C));
  ETXB_HOST_CU(etxb_host_smem(k, (int)cfg.dynamicSmemBytes, device, ready[which]));
  ETXB_HOST_CU(cudaLaunchKernelExC(&cfg, k, kargs));
  return ETXB_OK;
}
