// Drawing tokens: temperature, top-k, top-p and min-p over rows of logits, with given random numbers (etxb_sample).
//
// Mathematics.  The live tokens of a row (neither -inf nor NaN) stand in the order "larger logit first, equal logits by index".  Token r of that order
// has the weight w_r = exp((l_r - l_0) / T).  Every cut keeps a beginning of the order:
//   top-k   the first min(k, live)                                          mass W_k = the sum of their weights
//   top-p   those with (sum of the weights before r) < p * W_k
//   min-p   those with w_r >= min_p
// so together they keep the first n (at least one).  Drawn is the first token whose inclusive sum exceeds u * W_n.
//
// The sums have to be right next to every border, and the order of atomics must not change them: weights are integers, exp in 64 bits times 2^S with
// S = 62 - ceil(log2 V), so a row's sum fits 63 bits, is exact, and a weight is off by 2^-(S+1) <= 2^-43 of the largest.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdio.h>
#include <string.h>

#include "etxb_host.h"

namespace etxb_draw {

constexpr int THREADS = 1024, WARPS = THREADS / 32, BINS = 2048;

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
  return d < 0.0 ? exp(d * r.inv_t) : 1.0;
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

// What a lookup asks for: the token of a rank; the last token with less than `x` before it; the first with more than `x` up to it.
enum { BY_RANK, BY_MASS_BEFORE, BY_MASS_UPTO };
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
    bool hit;
    if (how == BY_RANK) hit = cb <= rank && rank < cb + c[k];
    else if (how == BY_MASS_BEFORE) hit = c[k] && (double)mb < x && (double)(mb + m[k]) >= x;
    else hit = (double)mb <= x && (double)(mb + m[k]) > x;
    if (hit) { s.bin = (uint32_t)(nbins - 1 - (2 * t + k)); s.before_count = cb; s.before_mass = mb; s.count = c[k]; }
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
  const void* k = a.dtype == ETXB_F32 ? (const void*)rows_kernel<float> : a.dtype == ETXB_F16 ? (const void*)rows_kernel<__half> : (const void*)rows_kernel<__nv_bfloat16>;
  ETXB_HOST_CU(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Shared)));
  void* kargs[] = {(void*)&a};
  ETXB_HOST_CU(cudaLaunchKernel(k, dim3((unsigned)a.rows), dim3(THREADS), kargs, sizeof(Shared), (cudaStream_t)cuda_stream));
  return ETXB_OK;
}
