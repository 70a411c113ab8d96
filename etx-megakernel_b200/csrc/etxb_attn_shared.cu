// Decode attention of one layer for sequences that share a prefix (etxb_attn_shared): a group of sequences has one block table for the positions
// they have in common and each sequence one for its own.
//
//   out_b,h = sum_i p_i v_i / sum_i p_i,  p_i = exp(scale * q_b,h . k_i - m),  i over the prefix of b's group and b's own positions
#include <cuda_bf16.h>
#include <stdio.h>
#include <string.h>

#include "etxb_host.h"

namespace etxb_shared {

constexpr int BS = 16;

struct Groups { int32_t first[ETXB_SHARED_MAX_SEQS + 1]; };

// A block takes one (sequence, q head); its warps take pages in turn.
constexpr int THREADS = 128, WARPS = 4;
__global__ void __launch_bounds__(THREADS) simple_kernel(const etxb_attn_shared_args a, const __grid_constant__ Groups groups) {
  __shared__ float q[256], o[WARPS][256], ml[WARPS][2];
  __shared__ int bad;
  const int b = blockIdx.x, head = blockIdx.y, G = a.NH / a.NKV, h = head / G, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, HD = a.HD;
  int g = 0;
  while (groups.first[g + 1] <= b) ++g;
  if (tid == 0) bad = 0;
  for (int i = tid; i < HD; i += THREADS) q[i] = __bfloat162float(((const __nv_bfloat16*)a.q)[b * a.q_stride + head * HD + i]) * a.scale;
  __syncthreads();
  float m = -INFINITY, l = 0.f, acc[8];
  for (int j = 0; j < 8; ++j) acc[j] = 0.f;
  for (int part = 0; part < 2; ++part) {
    const int32_t* table = part == 0 ? a.prefix_tables + g * a.prefix_stride : a.tables + b * a.table_stride;
    const int width = part == 0 ? a.prefix_width : a.table_width;
    const int len = part == 0 ? a.prefix_lens[g] : a.lens[b];
    if (len < 0 || len > width * BS) { atomicOr(&bad, ETXB_SHARED_BAD_LENGTH); continue; }
    for (int pg = warp; pg * BS < len; pg += WARPS) {
      const int page = table[pg], n = min(BS, len - pg * BS);
      if (page < 0 || page >= a.pages) { atomicOr(&bad, ETXB_SHARED_BAD_PAGE); continue; }
      const __nv_bfloat16* K = (const __nv_bfloat16*)a.kc + page * a.k_stride + (long long)h * HD * BS;
      const __nv_bfloat16* V = (const __nv_bfloat16*)a.vc + page * a.v_stride + (long long)h * HD * BS;
      const int pos = lane & 15;
      float s = 0.f;
      for (int c = lane >> 4; c < HD / 8; c += 2)
        for (int e = 0; e < 8; ++e) s = fmaf(q[c * 8 + e], __bfloat162float(K[(c * BS + pos) * 8 + e]), s);
      s += __shfl_xor_sync(~0u, s, 16);
      if (pos >= n) s = -INFINITY;
      float mx = s;
      for (int x = 8; x; x >>= 1) { const float y = __shfl_xor_sync(~0u, mx, x); mx = (mx >= y || mx != mx) ? mx : y; }
      const float mn = fmaxf(m, mx), f = m == -INFINITY ? 0.f : expf(m - mn);
      float p = pos < n && !(s == -INFINITY) ? expf(s - mn) : 0.f;
      m = mn; l *= f;
      for (int j = 0; j < 8; ++j) acc[j] *= f;
      for (int i = 0; i < n; ++i) {
        const float pi = __shfl_sync(~0u, p, i);
        l += pi;
        for (int j = 0; j < 8; ++j) if (lane + 32 * j < HD) acc[j] = fmaf(pi, __bfloat162float(V[(lane + 32 * j) * BS + i]), acc[j]);
      }
    }
  }
  if (lane == 0) { ml[warp][0] = m; ml[warp][1] = l; }
  for (int j = 0; j < 8; ++j) if (lane + 32 * j < HD) o[warp][lane + 32 * j] = acc[j];
  __syncthreads();
  float M = -INFINITY, L = 0.f;
  for (int w = 0; w < WARPS; ++w) M = fmaxf(M, ml[w][0]);
  // (a warp whose scores are all NaN has no maximum, but a sum that is NaN)
  for (int w = 0; w < WARPS; ++w) if (ml[w][1] != 0.f) L += ml[w][1] * (ml[w][0] == M ? 1.f : expf(ml[w][0] - M));
  for (int i = tid; i < HD; i += THREADS) {
    float y = 0.f;
    for (int w = 0; w < WARPS; ++w) if (ml[w][1] != 0.f) y = fmaf(o[w][i], ml[w][0] == M ? 1.f : expf(ml[w][0] - M), y);
    y = bad ? NAN : L == 0.f ? 0.f : y / L;
    ((__nv_bfloat16*)a.out)[b * a.out_stride + head * HD + i] = __float2bfloat16_rn(y);
  }
  if (bad && tid == 0 && a.status) atomicOr(a.status, bad);
}

static const char* check(const etxb_attn_shared_args& a) {
  if (a.NKV < 1 || a.NH < a.NKV || a.NH % a.NKV || a.NH / a.NKV > 16) return "NH a multiple of NKV, at most 16 q heads per kv head";
  if (a.HD < 16 || a.HD > 256 || a.HD % 16) return "head_dim a multiple of 16, at most 256";
  if (a.seqs < 0 || a.seqs > ETXB_SHARED_MAX_SEQS || a.groups < 0 || a.groups > ETXB_SHARED_MAX_SEQS) return "at most 1024 sequences and groups";
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
  if (a.group_first[0] != 0 || a.group_first[a.groups] != a.seqs) return "the groups cover the sequences in order";
  for (int g = 0; g < a.groups; ++g) if (a.group_first[g + 1] < a.group_first[g]) return "the groups cover the sequences in order";
  return nullptr;
}
static int32_t refuse(int32_t code, const char* why) {
  char m[200];
  snprintf(m, sizeof m, "attn_shared: %s", why);
  return etxb_host_fail(code, m);
}

}  // namespace etxb_shared

extern "C" int32_t etxb_attn_shared_work(int device, const etxb_attn_shared_args* args, size_t bytes, size_t* work_bytes) {
  using namespace etxb_shared;
  if (!args || bytes != sizeof(etxb_attn_shared_args) || !work_bytes) return refuse(ETXB_E_ARG, "needs an etxb_attn_shared_args");
  if (device < 0 || device >= 64) return refuse(ETXB_E_ARG, "device index out of range");
  if (const char* why = check(*args)) return refuse(ETXB_E_UNSUPPORTED, why);
  *work_bytes = 0;
  return ETXB_OK;
}

extern "C" int32_t etxb_attn_shared(int device, const etxb_attn_shared_args* args, size_t bytes, void* cuda_stream) {
  using namespace etxb_shared;
  if (!args || bytes != sizeof(etxb_attn_shared_args)) return refuse(ETXB_E_ARG, "needs an etxb_attn_shared_args");
  if (device < 0 || device >= 64) return refuse(ETXB_E_ARG, "device index out of range");
  if (const char* why = check(*args)) return refuse(ETXB_E_UNSUPPORTED, why);
  if (args->reserved != 0) return refuse(ETXB_E_ARG, "reserved is 0");
  if (args->seqs == 0) return ETXB_OK;
  if (const char* why = check_pointers(*args)) return refuse(ETXB_E_ARG, why);
  size_t need = 0;
  if (int32_t rc = etxb_attn_shared_work(device, args, bytes, &need)) return rc;
  if (need && (!args->work || args->work_bytes < need || ((uintptr_t)args->work & 255))) return refuse(ETXB_E_ARG, "work: as many bytes as etxb_attn_shared_work asks for, at a multiple of 256");
  Groups gr;
  memset(&gr, 0, sizeof gr);
  memcpy(gr.first, args->group_first, (size_t)(args->groups + 1) * 4);
  etxb_attn_shared_args a = *args;
  a.group_first = nullptr;
  EtxbDeviceScope scope(device);
  ETXB_HOST_CU(scope.err);
  simple_kernel<<<dim3((unsigned)a.seqs, (unsigned)a.NH), THREADS, 0, (cudaStream_t)cuda_stream>>>(a, gr);
  ETXB_HOST_CU(cudaGetLastError());
  return ETXB_OK;
}
