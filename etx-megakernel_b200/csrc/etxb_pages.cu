// Pages of a paged KV cache (etxb_pages_update): pages copied within a pool or between two, and the block tables that name them brought up to date, in
// one launch.  What is copied where is a list on the host: it is checked there, travels as a kernel parameter and needs no device memory of its own.
//
// Bound: HBM.  Every page is read once and written once (the copies of one page into several read it from L2).  A block takes one page of one layer and
// one tensor at a time; its threads hold four 16-byte pieces each, so a page of 16 KB is in flight at once.
// 257 pages of 24 layers, keys and values of 8 heads of 128: 404 MB read and written in 124 us, 6.5 TB/s, as fast as a plain copy; with the host's part, 257 pairs
// checked and handed over, 133 us a call.  A fork of 1037 positions into 8 sequences is 8 us a call, nearly all of it the launch.
// A copy of few pages is 39 us a call, 2 pages of 48 layers as 60: the checks of two pools of tensors in Python (a pool's own calls made them once).
#include <stdio.h>
#include <string.h>

#include <algorithm>
#include <mutex>
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
  int32_t n_move;                              // n_copy, or 0 where the pairs are there for the renumbering alone
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
  const long long units = (long long)h.n_move * h.layers * h.n_tensors;
  for (long long u = blockIdx.x; u < units; u += gridDim.x) {
    const int pair = (int)(u % h.n_move);
    const long long lt = u / h.n_move;
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
  const long long units = (long long)h.n_move * h.layers * h.n_tensors;
  const long long entries = std::max<long long>(h.n_set, (long long)h.n_share * h.shared);
  const long long blocks = std::max(std::max(units, (entries + THREADS - 1) / THREADS), (long long)h.n_remap);
  const int grid = (int)std::max<long long>(1, std::min<long long>(blocks, (long long)sms * 8));
  return data.size() <= SMALL ? launch<SMALL>(h, data.data(), data.size(), grid, st) : launch<LARGE>(h, data.data(), data.size(), grid, st);
}

// Pages of one tensor, layer by layer, from an address on.
struct Area {
  uintptr_t at;
  int64_t layer, page, bytes;
  int32_t layers, pages;
  int64_t extent() const { return page * (pages - 1) + bytes; }      // of a layer
  int64_t size() const { return (layers > 1 ? layer * (layers - 1) : 0) + extent(); }
};
// Whether two areas have no byte in common, where that is told by what they span, by their layers lying between each other's (views [layers][2][pages]) or by
// their pages doing so (views [layers][pages][2]).  Others that are apart by chance count as overlapping.
static bool apart(const Area& x, const Area& y) {
  if (x.at + x.size() <= y.at || y.at + y.size() <= x.at) return true;
  auto between = [&](int64_t step, int64_t first, int64_t second) {  // pieces of `first` and `second` bytes, every `step` bytes in both
    const int64_t d = (((int64_t)(y.at - x.at)) % step + step) % step;
    return d >= first && d + second <= step;
  };
  const bool one = x.layers == 1, layers = one || x.layer == y.layer;
  if (!one && layers && between(x.layer, x.extent(), y.extent())) return true;
  return x.page == y.page && layers && (one || x.layer % x.page == 0) && between(x.page, x.bytes, y.bytes);
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
  // (all tensors are copied at once, in no order: what one reads or writes no other one writes)
  for (int i = 0; a.n_copy && i < a.n_tensors; ++i) {
    const etxb_page_tensor& t = a.t[i];
    const Area to = {(uintptr_t)t.dst, t.dst_layer, t.dst_page, t.page_bytes, a.layers, a.dst_pages};
    for (int k = 0; k < a.n_tensors; ++k) {
      if (k == i) continue;
      const etxb_page_tensor& o = a.t[k];
      if (!apart(to, {(uintptr_t)o.src, o.src_layer, o.src_page, o.page_bytes, a.layers, a.src_pages}) ||
          !apart(to, {(uintptr_t)o.dst, o.dst_layer, o.dst_page, o.page_bytes, a.layers, a.dst_pages})) return "tensors overlap";
    }
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
    do {                                       // (once, but for a renumbering of many rows: the pages move with its first part)
      h.n_move = m == 0 ? h.n_copy : 0;
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
    ETXB_HOST_CU(etxb_host_sms(device, &sms));
    ETXB_HOST_CU(etxb_pages::run_all(*args, sms, (cudaStream_t)cuda_stream));
  } catch (const std::bad_alloc&) {
    return etxb_host_fail(ETXB_E_ARG, "pages: the lists do not fit the host's memory");
  }
  return ETXB_OK;
}

// ---- the books of a pool -------------------------------------------------------------------------------------------
struct etxb_pool {
  int device = 0, page_len = 16;
  etxb_pages_args base{};                       // the pool as source and destination, its tables
  etxb_pages_fn update = nullptr;
  std::mutex mutex;
  std::vector<int32_t> users;                   // sequences that hold a page
  int32_t n_free = 0, lowest = 0;               // free pages, and a page below which none is
  std::vector<std::vector<int32_t>> pages;      // of a row, in order
  std::vector<int32_t> length;                  // -1: no sequence
};

namespace etxb_pages {

static int32_t refuse(int32_t code, const char* fmt, long long x = 0, long long y = 0, long long z = 0) {
  char m[160], text[200];
  snprintf(m, sizeof m, fmt, x, y, z);
  snprintf(text, sizeof text, "pool: %s", m);
  return etxb_host_fail(code, text);
}
// One call on a pool: excludes others, and turns what the host's memory refuses into a status.
template <typename F>
static int32_t with(etxb_pool* p, F f) {
  if (!p) return refuse(ETXB_E_ARG, "null");
  try {
    std::lock_guard<std::mutex> lock(p->mutex);
    return f(*p);
  } catch (const std::exception&) {
    return refuse(ETXB_E_ARG, "the books do not fit the host's memory");
  }
}
static bool holds(const etxb_pool& p, int32_t row) { return row >= 0 && row < (int32_t)p.length.size() && p.length[(size_t)row] >= 0; }
static int32_t need(const etxb_pool& p, int32_t length) { return (int32_t)(((long long)length + p.page_len - 1) / p.page_len); }
// n free pages, the lowest first (nothing is marked yet)
static int32_t take(const etxb_pool& p, long long n, std::vector<int32_t>& out) {
  if (n > p.n_free) return refuse(ETXB_E_FULL, "%lld free pages, %lld are needed", p.n_free, n);
  out.reserve((size_t)n);
  for (int32_t i = p.lowest; (long long)out.size() < n; ++i) if (p.users[(size_t)i] == 0) out.push_back(i);
  return ETXB_OK;
}
static int32_t free_rows(const etxb_pool& p, int32_t n, std::vector<int32_t>& out) {
  for (int32_t r = 0; r < (int32_t)p.length.size() && (int32_t)out.size() < n; ++r) if (p.length[(size_t)r] < 0) out.push_back(r);
  return (int32_t)out.size() < n ? refuse(ETXB_E_FULL, "%lld free rows in the tables, %lld are needed", (long long)out.size(), n) : ETXB_OK;
}
static void hold(etxb_pool& p, const std::vector<int32_t>& fresh) {
  for (int32_t i : fresh) p.users[(size_t)i] = 1;
  p.n_free -= (int32_t)fresh.size();
  if (!fresh.empty() && fresh.front() == p.lowest) p.lowest = fresh.back() + 1;      // (they were the lowest free ones)
}
// (The books change once, when the call is made: replayed, it would write pages that are others' by then.)
static int32_t carry_out(etxb_pool& p, etxb_pages_args& a, void* stream) {
  if (p.update == etxb_pages_update) {
    cudaStreamCaptureStatus captured = cudaStreamCaptureStatusNone;
    ETXB_HOST_CU(cudaStreamIsCapturing((cudaStream_t)stream, &captured));
    if (captured != cudaStreamCaptureStatusNone) return refuse(ETXB_E_ARG, "calls that change the books are not captured");
  }
  return p.update(p.device, &a, sizeof a, stream);
}
static int32_t rows_once(const etxb_pool& p, const int32_t* rows, int32_t n) {
  if (n < 0 || (n && !rows)) return refuse(ETXB_E_ARG, "a list is null");
  std::vector<uint8_t> seen(p.length.size(), 0);
  for (int32_t i = 0; i < n; ++i) {
    if (!holds(p, rows[i])) return refuse(ETXB_E_ARG, "row %lld holds no sequence", rows[i]);
    if (seen[(size_t)rows[i]]) return refuse(ETXB_E_ARG, "each row once");
    seen[(size_t)rows[i]] = 1;
  }
  return ETXB_OK;
}

}  // namespace etxb_pages

extern "C" int32_t etxb_pool_create(int device, const etxb_pages_args* layout, size_t bytes, int32_t page_len, etxb_pages_fn update, etxb_pool** out) {
  using namespace etxb_pages;
  if (!out || !layout || bytes != sizeof(etxb_pages_args)) return refuse(ETXB_E_ARG, "needs an etxb_pages_args");
  if (page_len < 1 || layout->dst_pages < 1 || layout->table_rows < 1 || layout->table_width < 1) return refuse(ETXB_E_ARG, "at least one page, row, entry and position");
  if (layout->tables && layout->table_rows > 1 && layout->table_stride < layout->table_width) return refuse(ETXB_E_ARG, "rows of the tables overlap");
  if (device < 0 || device >= 64) return refuse(ETXB_E_ARG, "device index out of range");
  try {
    etxb_pool* p = new etxb_pool;
    p->device = device; p->page_len = page_len; p->update = update ? update : etxb_pages_update;
    p->base = *layout;
    for (etxb_page_tensor& t : p->base.t) { t.src = t.dst; t.src_layer = t.dst_layer; t.src_page = t.dst_page; }
    p->base.src_pages = layout->dst_pages;
    p->base.n_copy = p->base.n_set = p->base.n_share = p->base.n_remap = 0;
    p->users.assign((size_t)layout->dst_pages, 0);
    p->n_free = layout->dst_pages;
    p->pages.resize((size_t)layout->table_rows);
    p->length.assign((size_t)layout->table_rows, -1);
    *out = p;
  } catch (const std::exception&) {
    return refuse(ETXB_E_ARG, "the books do not fit the host's memory");
  }
  return ETXB_OK;
}

extern "C" int32_t etxb_pool_destroy(etxb_pool* pool) {
  delete pool;
  return ETXB_OK;
}

extern "C" int32_t etxb_pool_open(etxb_pool* pool, int32_t length, int32_t* row, void* cuda_stream) {
  using namespace etxb_pages;
  return with(pool, [&](etxb_pool& p) -> int32_t {
    if (!row || length < 0) return refuse(ETXB_E_ARG, "a length of %lld positions", length);
    const int32_t n = need(p, length);
    if (n > p.base.table_width) return refuse(ETXB_E_ARG, "%lld positions take %lld pages, a table has %lld", length, n, p.base.table_width);
    std::vector<int32_t> r, fresh;
    if (int32_t rc = free_rows(p, 1, r)) return rc;
    if (int32_t rc = take(p, n, fresh)) return rc;
    std::vector<int32_t> rows((size_t)n, r[0]), cols((size_t)n);
    for (int32_t i = 0; i < n; ++i) cols[(size_t)i] = i;
    std::vector<int32_t> mine = fresh;
    if (n) {
      etxb_pages_args a = p.base;
      a.n_set = n; a.set_rows = rows.data(); a.set_cols = cols.data(); a.set_pages = fresh.data();
      if (int32_t rc = carry_out(p, a, cuda_stream)) return rc;
    }
    hold(p, fresh);
    p.pages[(size_t)r[0]].swap(mine);
    p.length[(size_t)r[0]] = length;
    *row = r[0];
    return ETXB_OK;
  });
}

extern "C" int32_t etxb_pool_extend(etxb_pool* pool, const int32_t* rows, const int32_t* lengths, int32_t n, void* cuda_stream) {
  using namespace etxb_pages;
  return with(pool, [&](etxb_pool& p) -> int32_t {
    if (int32_t rc = rows_once(p, rows, n)) return rc;
    if (n && !lengths) return refuse(ETXB_E_ARG, "a list is null");
    long long more = 0;
    for (int32_t i = 0; i < n; ++i) {
      const int32_t have = p.length[(size_t)rows[i]], want = need(p, lengths[i]);
      if (lengths[i] < have) return refuse(ETXB_E_ARG, "row %lld has %lld positions, not %lld", rows[i], have, lengths[i]);
      if (want > p.base.table_width) return refuse(ETXB_E_ARG, "%lld positions take %lld pages, a table has %lld", lengths[i], want, p.base.table_width);
      more += want - (int32_t)p.pages[(size_t)rows[i]].size();
    }
    std::vector<int32_t> fresh, r, c;
    if (int32_t rc = take(p, more, fresh)) return rc;
    r.reserve(fresh.size()); c.reserve(fresh.size());
    for (int32_t i = 0; i < n; ++i) {
      std::vector<int32_t>& mine = p.pages[(size_t)rows[i]];
      mine.reserve((size_t)need(p, lengths[i]));
      for (int32_t k = (int32_t)mine.size(); k < need(p, lengths[i]); ++k) { r.push_back(rows[i]); c.push_back(k); }
    }
    if (!fresh.empty()) {
      etxb_pages_args a = p.base;
      a.n_set = (int32_t)fresh.size(); a.set_rows = r.data(); a.set_cols = c.data(); a.set_pages = fresh.data();
      if (int32_t rc = carry_out(p, a, cuda_stream)) return rc;
    }
    hold(p, fresh);
    for (size_t i = 0; i < fresh.size(); ++i) p.pages[(size_t)r[i]].push_back(fresh[i]);
    for (int32_t i = 0; i < n; ++i) p.length[(size_t)rows[i]] = lengths[i];
    return ETXB_OK;
  });
}

extern "C" int32_t etxb_pool_fork(etxb_pool* pool, int32_t row, int32_t n, int32_t length, int32_t* rows, void* cuda_stream) {
  using namespace etxb_pages;
  return with(pool, [&](etxb_pool& p) -> int32_t {
    if (!holds(p, row)) return refuse(ETXB_E_ARG, "row %lld holds no sequence", row);
    const int32_t have = p.length[(size_t)row], len = length == -1 ? have : length;
    if (n < 0 || (n && !rows) || len < 0 || len > have) return refuse(ETXB_E_ARG, "fork: %lld sequences from %lld positions of %lld", n, len, have);
    const int32_t full = len / p.page_len, part = len % p.page_len ? 1 : 0;
    std::vector<int32_t> r, fresh;
    if (int32_t rc = free_rows(p, n, r)) return rc;
    if (int32_t rc = take(p, (long long)n * part, fresh)) return rc;
    const std::vector<int32_t>& mine = p.pages[(size_t)row];
    std::vector<std::vector<int32_t>> theirs((size_t)n);
    for (int32_t i = 0; i < n; ++i) {
      theirs[(size_t)i].reserve((size_t)(full + part));
      theirs[(size_t)i].assign(mine.begin(), mine.begin() + full);
      if (part) theirs[(size_t)i].push_back(fresh[(size_t)i]);
    }
    if (n && (full || part)) {
      etxb_pages_args a = p.base;
      const std::vector<int32_t> src((size_t)n, part ? mine[(size_t)full] : 0), cols((size_t)n, full);
      if (part) {
        a.n_copy = n; a.src_ids = src.data(); a.dst_ids = fresh.data();
        a.n_set = n; a.set_rows = r.data(); a.set_cols = cols.data(); a.set_pages = fresh.data();
      }
      a.n_share = n; a.share_rows = r.data(); a.share_from = row; a.shared = full;
      if (int32_t rc = carry_out(p, a, cuda_stream)) return rc;
    }
    for (int32_t i = 0; i < full; ++i) p.users[(size_t)mine[(size_t)i]] += n;
    hold(p, fresh);
    for (int32_t i = 0; i < n; ++i) {
      p.pages[(size_t)r[(size_t)i]].swap(theirs[(size_t)i]);
      p.length[(size_t)r[(size_t)i]] = len;
      rows[i] = r[(size_t)i];
    }
    return ETXB_OK;
  });
}

extern "C" int32_t etxb_pool_close(etxb_pool* pool, const int32_t* rows, int32_t n) {
  using namespace etxb_pages;
  return with(pool, [&](etxb_pool& p) -> int32_t {
    if (int32_t rc = rows_once(p, rows, n)) return rc;
    for (int32_t i = 0; i < n; ++i) {
      for (int32_t page : p.pages[(size_t)rows[i]])
        if (--p.users[(size_t)page] == 0) { ++p.n_free; p.lowest = std::min(p.lowest, page); }
      p.pages[(size_t)rows[i]].clear();
      p.length[(size_t)rows[i]] = -1;
    }
    return ETXB_OK;
  });
}

extern "C" int32_t etxb_pool_compact(etxb_pool* pool, int32_t* moved, void* cuda_stream) {
  using namespace etxb_pages;
  return with(pool, [&](etxb_pool& p) -> int32_t {
    const int32_t total = (int32_t)p.users.size(), used = total - p.n_free;
    std::vector<int32_t> high, low;
    for (int32_t i = total - 1; i >= used; --i) if (p.users[(size_t)i]) high.push_back(i);
    for (int32_t i = p.lowest; i < used; ++i) if (!p.users[(size_t)i]) low.push_back(i);
    if (moved) *moved = (int32_t)high.size();
    if (high.empty()) return ETXB_OK;
    std::vector<int32_t> to((size_t)total, -1), rows, entries;
    for (size_t i = 0; i < high.size(); ++i) to[(size_t)high[i]] = low[i];
    for (int32_t r = 0; r < (int32_t)p.length.size(); ++r)
      if (!p.pages[(size_t)r].empty()) { rows.push_back(r); entries.push_back((int32_t)p.pages[(size_t)r].size()); }
    etxb_pages_args a = p.base;
    a.n_copy = (int32_t)high.size(); a.src_ids = high.data(); a.dst_ids = low.data();
    a.n_remap = (int32_t)rows.size(); a.remap_rows = rows.data(); a.remap_entries = entries.data();
    if (int32_t rc = carry_out(p, a, cuda_stream)) return rc;
    for (size_t i = 0; i < high.size(); ++i) { p.users[(size_t)low[i]] = p.users[(size_t)high[i]]; p.users[(size_t)high[i]] = 0; }
    for (int32_t r : rows)
      for (int32_t& page : p.pages[(size_t)r]) if (to[(size_t)page] >= 0) page = to[(size_t)page];
    p.lowest = used;
    return ETXB_OK;
  });
}

extern "C" int32_t etxb_pool_row(etxb_pool* pool, int32_t row, int32_t* length, int32_t* pages, int32_t capacity, int32_t* n) {
  using namespace etxb_pages;
  return with(pool, [&](etxb_pool& p) -> int32_t {
    if (row < 0 || row >= (int32_t)p.length.size() || capacity < 0) return refuse(ETXB_E_ARG, "row %lld of %lld", row, (long long)p.length.size());
    const std::vector<int32_t>& mine = p.pages[(size_t)row];
    if (length) *length = p.length[(size_t)row];
    if (n) *n = (int32_t)mine.size();
    if (pages) std::copy(mine.begin(), mine.begin() + std::min((size_t)capacity, mine.size()), pages);
    return ETXB_OK;
  });
}

extern "C" int32_t etxb_pool_free(etxb_pool* pool, int32_t* pages) {
  using namespace etxb_pages;
  return with(pool, [&](etxb_pool& p) -> int32_t {
    if (!pages) return refuse(ETXB_E_ARG, "null");
    *pages = p.n_free;
    return ETXB_OK;
  });
}
