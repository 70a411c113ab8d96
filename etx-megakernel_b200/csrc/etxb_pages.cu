// Pages of a paged KV cache (etxb_pages_update): pages copied within a pool or between two, and the block tables that name them brought up to date, in
// one launch.  What is copied where is a list on the host: it is checked there, travels as a kernel parameter and needs no device memory of its own.
//
// Bound: HBM.  Every page is read once and written once (the copies of one page into several read it from L2).  A block takes one page of one layer and
// one tensor at a time; its threads hold four 16-byte pieces each, so a page of 16 KB is in flight at once.
#include <stdio.h>
#include <string.h>

#include <algorithm>
#include <new>
#include <vector>

#include "etxb_host.h"

namespace etxb_pages {

constexpr int THREADS = 256, PIECES = 4;

struct Head {
  etxb_page_tensor t[ETXB_PAGES_MAX_TENSORS];
  int32_t* tables;
  long long table_stride;
  int32_t n_tensors, layers;
  int32_t n_copy, n_set, n_share, n_remap;     // data: n_copy (src, dst) pairs -- ascending in src where there is a remap --, n_set (row, column, page)
  int32_t share_from, shared;                  // triples, n_share rows, n_remap (row, entries) pairs
};
template <int N>
struct Params {
  Head h;
  int32_t data[N];
};

__device__ __forceinline__ uint4 ld_page(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}

template <int N>
__global__ void __launch_bounds__(THREADS) update_kernel(const __grid_constant__ Params<N> p) {
  const Head& h = p.h;
  const int tid = threadIdx.x;
  const int32_t* sets = p.data + 2 * h.n_copy;
  const int32_t* shares = sets + 3 * h.n_set;
  const int32_t* remaps = shares + h.n_share;
  const long long at = (long long)blockIdx.x * THREADS + tid, step = (long long)gridDim.x * THREADS;
  for (long long i = at; i < h.n_set; i += step) h.tables[sets[3 * i] * h.table_stride + sets[3 * i + 1]] = sets[3 * i + 2];
  for (long long i = at; i < (long long)h.n_share * h.shared; i += step) {
    const long long r = i / h.shared, c = i - r * h.shared;
    h.tables[shares[r] * h.table_stride + c] = h.tables[h.share_from * h.table_stride + c];
  }
  for (int i = blockIdx.x; i < h.n_remap; i += gridDim.x) {
    int32_t* row = h.tables + remaps[2 * i] * h.table_stride;
    for (int c = tid; c < remaps[2 * i + 1]; c += THREADS) {
      const int32_t page = row[c];
      int lo = 0, hi = h.n_copy;               // the first pair whose source is not below the page
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (p.data[2 * mid] < page) lo = mid + 1; else hi = mid;
      }
      if (lo < h.n_copy && p.data[2 * lo] == page) row[c] = p.data[2 * lo + 1];
    }
  }
  const long long units = (long long)h.n_copy * h.layers * h.n_tensors;
  for (long long u = blockIdx.x; u < units; u += gridDim.x) {
    const int pair = (int)(u % h.n_copy);
    const long long lt = u / h.n_copy;
    const etxb_page_tensor& t = h.t[lt % h.n_tensors];
    const long long layer = lt / h.n_tensors;
    const uint4* s = (const uint4*)((const char*)t.src + layer * t.src_layer + p.data[2 * pair] * t.src_page);
    uint4* d = (uint4*)((char*)t.dst + layer * t.dst_layer + p.data[2 * pair + 1] * t.dst_page);
    const long long n = t.page_bytes >> 4;
    for (long long i = tid; i < n; i += THREADS * PIECES) {
      uint4 v[PIECES];
#pragma unroll
      for (int k = 0; k < PIECES; ++k) if (i + k * THREADS < n) v[k] = ld_page(s + i + k * THREADS);
#pragma unroll
      for (int k = 0; k < PIECES; ++k) if (i + k * THREADS < n) __stcs(d + i + k * THREADS, v[k]);
    }
  }
}

template <int N>
static cudaError_t launch(const Head& h, const int32_t* data, size_t n, int grid, cudaStream_t st) {
  static_assert(sizeof(Params<N>) <= 32764, "kernel parameters");
  Params<N> p;
  p.h = h;
  memcpy(p.data, data, n * 4);
  update_kernel<N><<<grid, THREADS, 0, st>>>(p);
  return cudaGetLastError();
}
constexpr int SMALL = 192, LARGE = 7900;

static cudaError_t run(const Head& h, const std::vector<int32_t>& data, int sms, cudaStream_t st) {
  const long long units = (long long)h.n_copy * h.layers * h.n_tensors;
  const long long entries = std::max<long long>(h.n_set, (long long)h.n_share * h.shared);
  const long long blocks = std::max(std::max(units, (entries + THREADS - 1) / THREADS), (long long)h.n_remap);
  const int grid = (int)std::max<long long>(1, std::min<long long>(blocks, (long long)sms * 8));
  return data.size() <= SMALL ? launch<SMALL>(h, data.data(), data.size(), grid, st) : launch<LARGE>(h, data.data(), data.size(), grid, st);
}

// 0 or the text of what is wrong
static const char* check(const etxb_pages_args& a) {
  if (a.n_tensors < 1 || a.n_tensors > ETXB_PAGES_MAX_TENSORS || a.layers < 1 || a.layers > 65535) return "1 .. 4 tensors of 1 .. 65535 layers";
  if (a.n_copy < 0 || a.n_set < 0 || a.n_share < 0 || a.n_remap < 0) return "a list of negative length";
  if ((a.n_copy && (!a.src_ids || !a.dst_ids)) || (a.n_set && (!a.set_rows || !a.set_cols || !a.set_pages)) || (a.n_share && !a.share_rows) ||
      (a.n_remap && (!a.remap_rows || !a.remap_entries))) return "a list is null";
  if (a.src_pages < 1 || a.dst_pages < 1) return "pools of at least one page";
  const bool tables = a.n_set || a.n_share || a.n_remap;
  if (tables && (!a.tables || ((uintptr_t)a.tables & 3) || a.table_rows < 1 || a.table_width < 1 || a.table_stride < a.table_width)) return "tables: a pointer, rows that do not overlap";
  if (a.n_remap && (a.n_set || a.n_share)) return "pages are renumbered in a call of its own";
  bool same = true;
  for (int i = 0; i < a.n_tensors; ++i) {
    const etxb_page_tensor& t = a.t[i];
    if (t.page_bytes < 16) return "pages of at least 16 bytes";
    if (!a.n_copy) continue;
    if (!t.src || !t.dst) return "a tensor is null";
    if (((uintptr_t)t.src | (uintptr_t)t.dst | (uintptr_t)t.src_layer | (uintptr_t)t.src_page | (uintptr_t)t.dst_layer | (uintptr_t)t.dst_page | (uintptr_t)t.page_bytes) & 15)
      return "addresses, strides and page sizes are multiples of 16 bytes";
    if (t.src_page < t.page_bytes || t.dst_page < t.page_bytes || (a.layers > 1 && (t.src_layer < t.src_page * (a.src_pages - 1) + t.page_bytes ||
        t.dst_layer < t.dst_page * (a.dst_pages - 1) + t.page_bytes))) return "pages or layers overlap";
    const uintptr_t s0 = (uintptr_t)t.src, s1 = s0 + (a.layers - 1) * t.src_layer + (a.src_pages - 1) * t.src_page + t.page_bytes;
    const uintptr_t d0 = (uintptr_t)t.dst, d1 = d0 + (a.layers - 1) * t.dst_layer + (a.dst_pages - 1) * t.dst_page + t.page_bytes;
    const bool one = t.src == t.dst && t.src_page == t.dst_page && (a.layers == 1 || t.src_layer == t.dst_layer);
    if (!one && s0 < d1 && d0 < s1) return "source and destination are one pool or apart";
    if (i == 0) same = one;
    if (one != same) return "source and destination are one pool for every tensor, or for none";
  }
  std::vector<uint8_t> taken(a.n_copy ? (size_t)a.dst_pages : 0, 0);
  for (int i = 0; i < a.n_copy; ++i) {
    if (a.src_ids[i] < 0 || a.src_ids[i] >= a.src_pages || a.dst_ids[i] < 0 || a.dst_ids[i] >= a.dst_pages) return "a page outside its pool";
    if (taken[(size_t)a.dst_ids[i]]) return "a page is written twice";
    taken[(size_t)a.dst_ids[i]] = 1;
  }
  if (same)
    for (int i = 0; i < a.n_copy; ++i)
      if (a.src_ids[i] < a.dst_pages && taken[(size_t)a.src_ids[i]]) return "a page is read and written";
  const int limit = a.dst_pages;
  std::vector<long long> cells;
  for (int i = 0; i < a.n_set; ++i) {
    if (a.set_rows[i] < 0 || a.set_rows[i] >= a.table_rows || a.set_cols[i] < 0 || a.set_cols[i] >= a.table_width) return "an entry outside the tables";
    if (a.set_pages[i] < 0 || a.set_pages[i] >= limit) return "a page outside its pool";
    cells.push_back((long long)a.set_rows[i] * a.table_width + a.set_cols[i]);
  }
  std::sort(cells.begin(), cells.end());
  if (std::adjacent_find(cells.begin(), cells.end()) != cells.end()) return "an entry is written twice";
  std::vector<uint8_t> rows(a.n_share || a.n_remap ? (size_t)a.table_rows : 0, 0);
  if (a.n_share && (a.share_from < 0 || a.share_from >= a.table_rows || a.shared < 0 || a.shared > a.table_width)) return "shared entries outside the tables";
  for (int i = 0; i < a.n_share; ++i) {
    const int r = a.share_rows[i];
    if (r < 0 || r >= a.table_rows || r == a.share_from || rows[(size_t)r]) return "rows that share: inside the tables, each once, not the row they share with";
    rows[(size_t)r] = 1;
  }
  if (a.n_share) {
    rows[(size_t)a.share_from] = 1;
    for (int i = 0; i < a.n_set; ++i)
      if (rows[(size_t)a.set_rows[i]] && a.set_cols[i] < a.shared) return "an entry is shared and written";
  }
  for (int i = 0; i < a.n_remap; ++i) {
    const int r = a.remap_rows[i];
    if (r < 0 || r >= a.table_rows || rows[(size_t)r] || a.remap_entries[i] < 0 || a.remap_entries[i] > a.table_width) return "renumbered rows: inside the tables, each once";
    rows[(size_t)r] = 1;
  }
  if (a.n_remap) {
    if (!same && a.n_copy) return "pages are renumbered within one pool";
    std::vector<int32_t> src(a.src_ids, a.src_ids + a.n_copy);
    std::sort(src.begin(), src.end());
    if (std::adjacent_find(src.begin(), src.end()) != src.end()) return "a renumbered page has one new number";
  }
  return nullptr;
}

// The lists in launches of up to LARGE words.  A renumbering goes over its rows once for every launch of copies: no new number is another's old one.
static cudaError_t run_all(const etxb_pages_args& a, int sms, cudaStream_t st) {
  Head h;
  memset(&h, 0, sizeof h);
  memcpy(h.t, a.t, sizeof h.t);
  h.tables = a.tables; h.table_stride = a.table_stride; h.n_tensors = a.n_tensors; h.layers = a.layers; h.share_from = a.share_from; h.shared = a.shared;
  std::vector<int32_t> order((size_t)a.n_copy);
  for (int i = 0; i < a.n_copy; ++i) order[(size_t)i] = i;
  if (a.n_remap) std::sort(order.begin(), order.end(), [&](int x, int y) { return a.src_ids[x] < a.src_ids[y]; });
  std::vector<int32_t> data;
  int c = 0, s = 0, r = 0;
  while (c < a.n_copy || s < a.n_set || r < a.n_share) {
    data.clear();
    const int room_c = a.n_remap ? LARGE / 4 : LARGE / 2;
    h.n_copy = std::min(a.n_copy - c, room_c);
    for (int i = 0; i < h.n_copy; ++i, ++c) { data.push_back(a.src_ids[order[(size_t)c]]); data.push_back(a.dst_ids[order[(size_t)c]]); }
    h.n_set = std::min(a.n_set - s, (int)((LARGE - data.size()) / 3));
    for (int i = 0; i < h.n_set; ++i, ++s) { data.push_back(a.set_rows[s]); data.push_back(a.set_cols[s]); data.push_back(a.set_pages[s]); }
    h.n_share = std::min(a.n_share - r, (int)(LARGE - data.size()));
    for (int i = 0; i < h.n_share; ++i, ++r) data.push_back(a.share_rows[r]);
    const size_t fixed = data.size();
    int m = 0;
    do {                                       // (once, but for a renumbering of many rows: the copies go with its first part)
      data.resize(fixed);
      h.n_remap = std::min(a.n_remap - m, (int)((LARGE - fixed) / 2));
      for (int i = 0; i < h.n_remap; ++i, ++m) { data.push_back(a.remap_rows[m]); data.push_back(a.remap_entries[m]); }
      const cudaError_t e = run(h, data, sms, st);
      if (e != cudaSuccess) return e;
    } while (m < a.n_remap);
  }
  return cudaSuccess;
}

}  // namespace etxb_pages

extern "C" int32_t etxb_pages_update(int device, const etxb_pages_args* args, size_t bytes, void* cuda_stream) {
  if (!args || bytes != sizeof(etxb_pages_args)) return etxb_host_fail(ETXB_E_ARG, "pages: needs an etxb_pages_args");
  if (device < 0 || device >= 64) return etxb_host_fail(ETXB_E_ARG, "pages: device index out of range");
  try {
    const char* why = etxb_pages::check(*args);
    if (why) {
      char m[200];
      snprintf(m, sizeof m, "pages: %s", why);
      return etxb_host_fail(ETXB_E_ARG, m);
    }
    if (!args->n_copy && !args->n_set && !(args->n_share && args->shared)) return ETXB_OK;
    EtxbDeviceScope scope(device);
    ETXB_HOST_CU(scope.err);
    int sms = 0;
    ETXB_HOST_CU(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
    ETXB_HOST_CU(etxb_pages::run_all(*args, sms, (cudaStream_t)cuda_stream));
  } catch (const std::bad_alloc&) {
    return etxb_host_fail(ETXB_E_ARG, "pages: the lists do not fit the host's memory");
  }
  return ETXB_OK;
}
