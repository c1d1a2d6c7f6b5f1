// Requests that go on from what others hold, gfx950: the page tables, lengths and
// free pages after row i has become a continuation of row parents[i], the pages
// that have to be copied for it, and the rows of a state taken along.
//
// Pages that a request has filled are never written again, so its continuations
// hold them in common (extra[page] counts the holders beyond the first).  The page
// that it is still filling stays with its first continuation and is copied for the
// others.  Whoever has no continuation gives up his pages; one that nobody holds any
// more goes back on the stack.
//
// Everything is whole numbers: atomics add up to the same whatever their order, and
// the order of pages on the stack is that of the rows and columns.
#include "common.h"
#include "mod_keys.h"

namespace hydra {
namespace {

constexpr int kThreads = 256;
constexpr int kWide = 1024;
constexpr int kMaxRows = 8192;  // counted in LDS

struct ForkArgs {
  const int* parents;
  int *lengths, *table, *free_pages, *free_count, *extra;
  int64_t table_rs;
  int *sources, *copies, *taken;   // results, [N]; taken: the row that each one continues, -1: none
  uint8_t* granted;
  // scratch: continuations and the first of them, [N]; lengths, tables and stack before;
  // the first place in the table, j P + c, of those that give a page up, and how many
  // pages each row puts back
  int *old_free, *kids, *first, *old_len, *back, *old_table, *owner;
  int N, P, F, pages, shift;
};

__device__ __forceinline__ bool is_page(const ForkArgs& a, int p) {
  return static_cast<unsigned>(p) < static_cast<unsigned>(a.pages);
}
// Pages that a row of `len` tokens has filled, and holds.
__device__ __forceinline__ int full_of(const ForkArgs& a, int len) { return len <= 0 ? 0 : min(len >> a.shift, a.P); }
__device__ __forceinline__ int held_of(const ForkArgs& a, int len) {
  const int full = full_of(a, len);
  return len > 0 && full < a.P && (len & ((1 << a.shift) - 1)) != 0 ? full + 1 : full;
}
__device__ __forceinline__ int parent_of(const ForkArgs& a, int i) {
  const int p = a.parents[i];
  return static_cast<unsigned>(p) < static_cast<unsigned>(a.N) ? p : -1;
}

__device__ __forceinline__ int block_incl_sum(int x, int* part, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int s = wave_incl_sum(x);
  __syncthreads();  // the last use of `part` is over
  if (lane == 63) part[wave] = s;
  __syncthreads();
  int all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    if (w < wave) s += part[w];
    all += part[w];
  }
  total = all;
  return s;
}

// Workgroup 0 counts the continuations in LDS; the others clear `owner`.
__global__ __launch_bounds__(kWide) void fork_count_kernel(ForkArgs a) {
  __shared__ int kids[kMaxRows], first[kMaxRows];
  const int tid = threadIdx.x;
  if (blockIdx.x > 0) {
    const int step = (gridDim.x - 1) * kWide;
    for (int64_t i = (blockIdx.x - 1) * kWide + tid; i < a.pages; i += step) a.owner[i] = a.N * a.P;
    return;
  }
  for (int i = tid; i < a.N; i += kWide) {
    kids[i] = 0;
    first[i] = a.N;
  }
  __syncthreads();
  for (int i = tid; i < a.N; i += kWide) {
    const int p = parent_of(a, i);
    if (p < 0) continue;
    atomicAdd(&kids[p], 1);
    atomicMin(&first[p], i);
  }
  __syncthreads();
  for (int i = tid; i < a.N; i += kWide) {
    a.kids[i] = kids[i];
    a.first[i] = first[i];
    a.old_len[i] = a.lengths[i];
  }
  if (tid == 0) {
    const int free = *a.free_count;
    *a.old_free = free < 0 ? 0 : (free > a.F ? a.F : free);
  }
}

// Row j's pages: kept before they are written over, and their holders counted.
__global__ __launch_bounds__(kThreads) void fork_share_kernel(ForkArgs a) {
  for (int j = blockIdx.x; j < a.N; j += gridDim.x) {
    const int len = a.old_len[j], full = full_of(a, len), held = held_of(a, len), kids = a.kids[j];
    for (int c = threadIdx.x; c < held; c += kThreads) {
      const int p = a.table[j * a.table_rs + c];
      a.old_table[static_cast<int64_t>(j) * a.P + c] = p;
      if (!is_page(a, p)) continue;
      if (c < full && kids > 1) atomicAdd(&a.extra[p], kids - 1);
      if (kids == 0) {
        atomicAdd(&a.extra[p], -1);
        atomicMin(&a.owner[p], j * a.P + c);
      }
    }
  }
}

// Whether column c of row j, which has no continuation, is the place to put the page back
// from.
__device__ __forceinline__ bool gives_back(const ForkArgs& a, int j, int c, int p) {
  return is_page(a, p) && a.owner[p] == j * a.P + c && a.extra[p] < 0;
}

__global__ __launch_bounds__(kThreads) void fork_back_kernel(ForkArgs a) {
  __shared__ int part[kThreads / 64];
  for (int j = blockIdx.x; j < a.N; j += gridDim.x) {
    const int held = a.kids[j] == 0 ? held_of(a, a.old_len[j]) : 0;
    int count = 0, all;
    for (int c = threadIdx.x; c < held; c += kThreads) count += gives_back(a, j, c, a.old_table[static_cast<int64_t>(j) * a.P + c]);
    block_incl_sum(count, part, all);
    if (threadIdx.x == 0) a.back[j] = all;
  }
}

// The sum of value(i), i < n, by the whole workgroup.
template <typename Value>
__device__ __forceinline__ int block_sum_upto(int n, int* part, Value&& value) {
  int mine = 0, all;
  for (int i = threadIdx.x; i < n; i += kThreads) mine += value(i);
  block_incl_sum(mine, part, all);
  return all;
}

__global__ __launch_bounds__(kThreads) void fork_push_kernel(ForkArgs a) {
  __shared__ int part[kThreads / 64];
  for (int j = blockIdx.x; j < a.N; j += gridDim.x) {
    if (a.back[j] == 0) continue;
    int64_t top = *a.old_free + static_cast<int64_t>(block_sum_upto(j, part, [&](int i) { return a.back[i]; }));
    const int held = held_of(a, a.old_len[j]);
    for (int c0 = 0; c0 < held; c0 += kThreads) {
      const int c = c0 + threadIdx.x, p = c < held ? a.old_table[static_cast<int64_t>(j) * a.P + c] : -1;
      const bool back = gives_back(a, j, c, p);
      int count;
      const int64_t to = top + block_incl_sum(back, part, count) - 1;
      if (back) {
        a.extra[p] = 0;
        if (to < a.F) a.free_pages[to] = p;
      }
      top += count;
    }
  }
}

// The page that row i has to get a copy of, or -1.
__device__ __forceinline__ int source_of(const ForkArgs& a, int i) {
  const int p = parent_of(a, i);
  if (p < 0 || a.first[p] == i) return -1;
  const int len = a.old_len[p], full = full_of(a, len);
  if (held_of(a, len) == full) return -1;
  const int page = a.old_table[static_cast<int64_t>(p) * a.P + full];
  return is_page(a, page) ? page : -1;
}

// Row i's new pages, each workgroup counting the copies before its own again.
__global__ __launch_bounds__(kThreads) void fork_take_kernel(ForkArgs a) {
  __shared__ int part[kThreads / 64];
  const int sum = block_sum_upto(a.N, part, [&](int i) { return a.back[i]; });
  const int free = static_cast<int>(min(static_cast<int64_t>(a.F), static_cast<int64_t>(*a.old_free) + sum));
  for (int i = blockIdx.x; i < a.N; i += gridDim.x) {
    const int p = parent_of(a, i), len = p >= 0 ? a.old_len[p] : 0, full = full_of(a, len);
    const int source = source_of(a, i);
    const bool need = source >= 0, last = i == a.N - 1;
    const int rank = need || last ? block_sum_upto(i, part, [&](int x) { return source_of(a, x) >= 0 ? 1 : 0; }) : 0;
    const bool granted = !need || rank < free;
    const int held = granted ? held_of(a, len) : 0, copy = need && granted ? a.free_pages[free - 1 - rank] : -1;
    const int* from = a.old_table + static_cast<int64_t>(p < 0 ? 0 : p) * a.P;
    for (int c = threadIdx.x; c < a.P; c += kThreads) {
      int e = c < held ? from[c] : -1;
      if (c == full && copy >= 0) e = copy;
      a.table[i * a.table_rs + c] = e;
    }
    if (!granted) {  // its share of the filled pages
      for (int c = threadIdx.x; c < full; c += kThreads)
        if (is_page(a, from[c])) atomicAdd(&a.extra[from[c]], -1);
    }
    if (threadIdx.x == 0) {
      a.lengths[i] = granted ? len : 0;
      a.granted[i] = granted;
      a.sources[i] = need && granted ? source : -1;
      a.copies[i] = copy;
      a.taken[i] = granted ? p : -1;
      if (last) *a.free_count = free - min(rank + (need ? 1 : 0), free);
    }
  }
}

// All of it by one workgroup, where rows and their tables are few: 4.6 us for 4 rows of 64
// pages.  In a graph with the copies and states of 2 rows of 16 pages 9.2 us (by the five
// kernels 14.9), 64 rows of 64 16.7 (19.2); 128 of 64 20.1 (19.8), where it still saves the
// host four launches.  What its threads hand each other through memory need not leave
// the XCD's L2: atomics, loads and fences are of the workgroup's scope.
constexpr int kSmallRows = 256, kSmallEntries = 8192;

__device__ __forceinline__ int seen(const int* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
}
__device__ __forceinline__ void put(int* p, int v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
}
__device__ __forceinline__ void add(int* p, int v) {
  __hip_atomic_fetch_add(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
}

// Inclusive sum over 1024 threads; `total` gets the whole sum.
__device__ __forceinline__ int wide_incl_sum(int x, int* part, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int s = wave_incl_sum(x);
  __syncthreads();
  if (lane == 63) part[wave] = s;
  __syncthreads();
  int all = 0;
#pragma unroll
  for (int w = 0; w < kWide / 64; ++w) {
    if (w < wave) s += part[w];
    all += part[w];
  }
  total = all;
  return s;
}

__global__ __launch_bounds__(kWide) void fork_small_kernel(ForkArgs a) {
  __shared__ int par[kSmallRows], len[kSmallRows], kids[kSmallRows], first[kSmallRows], copy[kSmallRows];
  __shared__ int old[kSmallEntries];
  __shared__ int part[kWide / 64];
  __shared__ bool ok[kSmallRows];
  const int tid = threadIdx.x, all = a.N * a.P;
  int free = *a.free_count;
  free = free < 0 ? 0 : (free > a.F ? a.F : free);
  if (tid < a.N) {
    par[tid] = parent_of(a, tid);
    len[tid] = a.lengths[tid];
    kids[tid] = 0;
    first[tid] = a.N;
  }
  __syncthreads();
  if (tid < a.N && par[tid] >= 0) {
    atomicAdd(&kids[par[tid]], 1);
    atomicMin(&first[par[tid]], tid);
  }
  for (int e = tid; e < all; e += kWide) {
    const int j = e / a.P, c = e - j * a.P;
    if (c >= held_of(a, len[j])) continue;
    old[e] = a.table[j * a.table_rs + c];
    if (is_page(a, old[e])) put(&a.owner[old[e]], all);
  }
  __threadfence_block();
  __syncthreads();
  for (int e = tid; e < all; e += kWide) {
    const int j = e / a.P, c = e - j * a.P;
    if (c >= held_of(a, len[j]) || !is_page(a, old[e])) continue;
    if (c < full_of(a, len[j]) && kids[j] > 1) add(&a.extra[old[e]], kids[j] - 1);
    if (kids[j] == 0) {
      add(&a.extra[old[e]], -1);
      __hip_atomic_fetch_min(&a.owner[old[e]], e, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    }
  }
  __threadfence_block();
  __syncthreads();
  for (int e0 = 0; e0 < all; e0 += kWide) {
    const int e = e0 + tid, j = e < all ? e / a.P : 0, c = e - j * a.P;
    const bool mine = e < all && kids[j] == 0 && c < held_of(a, len[j]) && is_page(a, old[e]);
    const bool back = mine && seen(&a.owner[old[e]]) == e && seen(&a.extra[old[e]]) < 0;
    int count;
    const int to = free + wide_incl_sum(back, part, count) - 1;
    if (back) {
      put(&a.extra[old[e]], 0);
      if (to < a.F) put(&a.free_pages[to], old[e]);
    }
    free = min(a.F, free + count);
  }
  __threadfence_block();
  __syncthreads();
  {
    int source = -1;
    if (tid < a.N && par[tid] >= 0 && first[par[tid]] != tid) {
      const int full = full_of(a, len[par[tid]]);
      if (held_of(a, len[par[tid]]) > full) source = old[par[tid] * a.P + full];
    }
    const bool need = is_page(a, source);
    int count;
    const int rank = wide_incl_sum(need, part, count) - 1;
    if (tid < a.N) {
      const bool granted = !need || rank < free;
      ok[tid] = granted;
      copy[tid] = need && granted ? seen(&a.free_pages[free - 1 - rank]) : -1;
      a.lengths[tid] = granted && par[tid] >= 0 ? len[par[tid]] : 0;
      a.granted[tid] = granted;
      a.sources[tid] = need && granted ? source : -1;
      a.copies[tid] = copy[tid];
      a.taken[tid] = granted ? par[tid] : -1;
    }
    if (tid == 0) *a.free_count = free - min(count, free);
  }
  __syncthreads();
  for (int e = tid; e < all; e += kWide) {
    const int i = e / a.P, c = e - i * a.P, p = par[i], n = p >= 0 ? len[p] : 0, full = full_of(a, n);
    const int held = held_of(a, n), from = c < held ? old[p * a.P + c] : -1;
    if (!ok[i] && c < full && is_page(a, from)) add(&a.extra[from], -1);  // its share of the filled pages
    a.table[i * a.table_rs + c] = !ok[i] ? -1 : (c == full && copy[i] >= 0 ? copy[i] : from);
  }
}

// Whole pages, sources[i] to copies[i], keys and values (and scales): pieces of V.
struct CopyArgs {
  const int *sources, *copies;
  char *p[4];
  int64_t page_st[4], h_st[4];    // bytes
  uint32_t row_st[4], pieces[4];  // bytes; pieces of a row
  int N, K, page, pages;
};

template <typename V>
__device__ __forceinline__ void copy_page(const CopyArgs& a, int t, int64_t from, int64_t to) {
  const uint32_t head = a.page * a.pieces[t], all = a.K * head;
  for (uint32_t e = blockIdx.x * kThreads + threadIdx.x; e < all; e += gridDim.x * kThreads) {
    const uint32_t h = e / head, x = e - h * head, r = x / a.pieces[t], c = x - r * a.pieces[t];
    char* at = a.p[t] + h * a.h_st[t] + static_cast<uint64_t>(r) * a.row_st[t] + c * static_cast<uint32_t>(sizeof(V));
    *reinterpret_cast<V*>(at + to * a.page_st[t]) = *reinterpret_cast<const V*>(at + from * a.page_st[t]);
  }
}

template <typename V>
__global__ __launch_bounds__(kThreads) void copy_pages_kernel(CopyArgs a) {
  for (int i = blockIdx.y; i < a.N; i += gridDim.y) {
    const int from = a.sources[i], to = a.copies[i];
    if (static_cast<unsigned>(from) >= static_cast<unsigned>(a.pages) ||
        static_cast<unsigned>(to) >= static_cast<unsigned>(a.pages))
      continue;
    copy_page<V>(a, 0, from, to);
    copy_page<V>(a, 1, from, to);
    if (a.p[2]) {
      copy_page<uint32_t>(a, 2, from, to);
      copy_page<uint32_t>(a, 3, from, to);
    }
  }
}

// x[i] = x[parents[i]] in place, rows of `pieces` of V.  A workgroup has a range of
// columns of all rows for itself: it reads what the rows get, waits, and writes.
// 1024 rows of 64 KB: 23.2 us, 5.8 TB/s both ways.
constexpr int kTakeThreads = 1024, kTakePieces = 8;

struct TakeArgs {
  char* x;
  const int* parents;
  int64_t row_st;      // bytes
  int64_t pieces;
  int N, cols, log;    // columns of a workgroup: a power of two
};

__device__ __forceinline__ void hold(uint4& v) { asm volatile("" : "+v"(v.x), "+v"(v.y), "+v"(v.z), "+v"(v.w)); }
__device__ __forceinline__ void hold(uint8_t& v) {
  uint32_t w = v;
  asm volatile("" : "+v"(w));
  v = static_cast<uint8_t>(w);
}

template <typename V>
__global__ __launch_bounds__(kTakeThreads) void take_rows_kernel(TakeArgs a) {
  const int64_t c0 = static_cast<int64_t>(blockIdx.x) << a.log;
  V v[kTakePieces];
#pragma unroll
  for (int u = 0; u < kTakePieces; ++u) {
    const int e = u * kTakeThreads + threadIdx.x, i = e >> a.log;
    const int64_t c = c0 + (e & (a.cols - 1));
    v[u] = V{};
    if (i >= a.N || c >= a.pieces) continue;
    const int p = a.parents[i];
    if (static_cast<unsigned>(p) >= static_cast<unsigned>(a.N) || p == i) continue;
    v[u] = *reinterpret_cast<const V*>(a.x + p * a.row_st + c * static_cast<int64_t>(sizeof(V)));
  }
  // the values are here before anybody writes
#pragma unroll
  for (int u = 0; u < kTakePieces; ++u) hold(v[u]);
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kTakePieces; ++u) {
    const int e = u * kTakeThreads + threadIdx.x, i = e >> a.log;
    const int64_t c = c0 + (e & (a.cols - 1));
    if (i >= a.N || c >= a.pieces) continue;
    const int p = a.parents[i];
    if (static_cast<unsigned>(p) >= static_cast<unsigned>(a.N) || p == i) continue;
    *reinterpret_cast<V*>(a.x + i * a.row_st + c * static_cast<int64_t>(sizeof(V))) = v[u];
  }
}

int page_shift(int64_t page_size) {
  for (int s = 4; s <= 12; ++s)
    if (page_size == (int64_t(1) << s)) return s;
  return -1;
}

int check_fork(int64_t N, int64_t P, int64_t pages) {
  HYDRA_REQUIRE(N >= 1 && P >= 1 && pages >= 1, "page_fork: bad size");
  HYDRA_REQUIRE(N <= kMaxRows, "page_fork: at most 8192 rows");
  HYDRA_REQUIRE(P < (int64_t(1) << 31) && N * P < (int64_t(1) << 31) && pages < (int64_t(1) << 31),
                "page_fork: too large");
  return HYDRA_OK;
}

int64_t scratch_bytes(int64_t N, int64_t P, int64_t pages) { return 4 * (1 + 4 * N + N * P + pages); }

}  // namespace
}  // namespace hydra

using namespace hydra;

extern "C" int hydra_page_fork_workspace(int64_t N, int64_t P, int64_t pages, int64_t* bytes) {
  const int rc = check_fork(N, P, pages);
  if (rc != HYDRA_OK) return rc;
  HYDRA_REQUIRE(bytes != nullptr, "page_fork_workspace: null pointer");
  *bytes = scratch_bytes(N, P, pages);
  return HYDRA_OK;
}

extern "C" int hydra_page_fork(const int* parents, int* lengths, int* table, int64_t table_rs, int* free_pages,
                               int64_t free_capacity, int* free_count, int* extra, int* sources, int* copies, int* taken,
                               void* granted, int64_t N, int64_t P, int64_t page_size, int64_t pages, void* workspace,
                               int64_t workspace_size, void* stream) {
  const int rc = check_fork(N, P, pages);
  if (rc != HYDRA_OK) return rc;
  const int shift = page_shift(page_size);
  HYDRA_REQUIRE(shift >= 0, "page_fork: page_size must be a power of two in [16, 4096]");
  HYDRA_REQUIRE(table_rs >= P, "page_fork: table row stride < columns");
  HYDRA_REQUIRE(P * page_size < (int64_t(1) << 31) && free_capacity >= 0 && free_capacity < (int64_t(1) << 31),
                "page_fork: too large");
  HYDRA_REQUIRE(parents && lengths && table && (free_pages || free_capacity == 0) && free_count && extra && sources &&
                    copies && taken && granted,
                "page_fork: null pointer");
  HYDRA_REQUIRE(workspace && reinterpret_cast<uintptr_t>(workspace) % 4 == 0 &&
                    workspace_size >= scratch_bytes(N, P, pages),
                "page_fork: workspace too small");
  ForkArgs a{};
  a.parents = parents;
  a.lengths = lengths;
  a.table = table;
  a.free_pages = free_pages;
  a.free_count = free_count;
  a.extra = extra;
  a.table_rs = table_rs;
  a.sources = sources;
  a.copies = copies;
  a.taken = taken;
  a.granted = static_cast<uint8_t*>(granted);
  a.old_free = static_cast<int*>(workspace);
  a.kids = a.old_free + 1;
  a.first = a.kids + N;
  a.old_len = a.first + N;
  a.back = a.old_len + N;
  a.old_table = a.back + N;
  a.owner = a.old_table + N * P;
  a.N = static_cast<int>(N);
  a.P = static_cast<int>(P);
  a.F = static_cast<int>(free_capacity);
  a.pages = static_cast<int>(pages);
  a.shift = shift;
  auto st = static_cast<hipStream_t>(stream);
  if (N <= kSmallRows && N * P <= kSmallEntries) {
    fork_small_kernel<<<1, kWide, 0, st>>>(a);
    return check_launch("page_fork");
  }
  const int64_t wide = (pages + kWide - 1) / kWide;
  const unsigned rows = static_cast<unsigned>(N);
  fork_count_kernel<<<static_cast<unsigned>(1 + (wide < 1024 ? wide : 1024)), kWide, 0, st>>>(a);
  fork_share_kernel<<<rows, kThreads, 0, st>>>(a);
  fork_back_kernel<<<rows, kThreads, 0, st>>>(a);
  fork_push_kernel<<<rows, kThreads, 0, st>>>(a);
  fork_take_kernel<<<rows, kThreads, 0, st>>>(a);
  return check_launch("page_fork");
}

extern "C" int hydra_page_copy(void* k_pages, void* v_pages, float* k_scales, float* v_scales, const int* sources,
                               const int* copies, int64_t N, int64_t Hkv, int64_t hd, int64_t pages, int64_t page_size,
                               const int64_t* kp_st, const int64_t* vp_st, const int64_t* ks_st, const int64_t* vs_st,
                               int element_size, void* stream) {
  HYDRA_REQUIRE(N >= 0 && Hkv >= 1 && hd >= 1 && pages >= 1, "page_copy: bad size");
  HYDRA_REQUIRE(page_shift(page_size) >= 0, "page_copy: page_size must be a power of two in [16, 4096]");
  HYDRA_REQUIRE(element_size == 1 || element_size == 2 || element_size == 4, "page_copy: elements of 1, 2 or 4 bytes");
  HYDRA_REQUIRE(N < (int64_t(1) << 31) && Hkv <= 65535 && hd <= 65536 && Hkv * hd * page_size < (int64_t(1) << 28) &&
                    pages < (int64_t(1) << 31),
                "page_copy: too large");
  if (N == 0) return HYDRA_OK;
  HYDRA_REQUIRE(k_pages && v_pages && sources && copies && kp_st && vp_st, "page_copy: null pointer");
  const bool scales = k_scales != nullptr;
  HYDRA_REQUIRE(scales == (v_scales != nullptr) && (!scales || (ks_st && vs_st)), "page_copy: null pointer");
  HYDRA_REQUIRE(kp_st[3] == 1 && vp_st[3] == 1 && (!scales || (ks_st[2] == 1 && vs_st[2] == 1)),
                "page_copy: rows need unit stride");
  CopyArgs a{};
  a.sources = sources;
  a.copies = copies;
  a.p[0] = static_cast<char*>(k_pages);
  a.p[1] = static_cast<char*>(v_pages);
  a.p[2] = reinterpret_cast<char*>(k_scales);
  a.p[3] = reinterpret_cast<char*>(v_scales);
  a.N = static_cast<int>(N);
  a.K = static_cast<int>(Hkv);
  a.page = static_cast<int>(page_size);
  a.pages = static_cast<int>(pages);
  const int64_t e = element_size;
  bool vec = hd * e % 16 == 0 && aligned16(k_pages) && aligned16(v_pages);
  for (int t = 0; t < 2; ++t) {
    const int64_t* s = t ? vp_st : kp_st;
    HYDRA_REQUIRE(s[2] >= 0 && s[2] < (int64_t(1) << 32) / e, "page_copy: rows too far apart");
    a.page_st[t] = s[0] * e;
    a.h_st[t] = s[1] * e;
    a.row_st[t] = static_cast<uint32_t>(s[2] * e);
    vec = vec && (a.page_st[t] | a.h_st[t] | (s[2] * e)) % 16 == 0;
  }
  for (int t = 0; t < 2; ++t) a.pieces[t] = static_cast<uint32_t>(vec ? hd * e / 16 : hd * e);
  for (int t = 2; t < 4 && scales; ++t) {
    const int64_t* s = t == 3 ? vs_st : ks_st;
    a.page_st[t] = s[0] * 4;
    a.h_st[t] = s[1] * 4;
    a.row_st[t] = 4;
    a.pieces[t] = 1;
  }
  const int64_t all = Hkv * page_size * a.pieces[0], wide = (all + kThreads - 1) / kThreads;
  const dim3 grid(static_cast<unsigned>(wide < 64 ? wide : 64), static_cast<unsigned>(N < 65535 ? N : 65535));
  auto st = static_cast<hipStream_t>(stream);
  if (vec) copy_pages_kernel<uint4><<<grid, kThreads, 0, st>>>(a);
  else copy_pages_kernel<uint8_t><<<grid, kThreads, 0, st>>>(a);
  return check_launch("page_copy");
}

extern "C" int hydra_rows_take(void* x, int64_t row_stride_bytes, int64_t row_bytes, const int* parents, int64_t N,
                               void* stream) {
  HYDRA_REQUIRE(N >= 0 && row_bytes >= 0, "rows_take: bad size");
  HYDRA_REQUIRE(N <= kTakeThreads * kTakePieces, "rows_take: at most 8192 rows");
  HYDRA_REQUIRE(row_bytes < (int64_t(1) << 40) && row_stride_bytes < (int64_t(1) << 40), "rows_take: too large");
  if (N <= 1 || row_bytes == 0) return HYDRA_OK;
  HYDRA_REQUIRE(x && parents, "rows_take: null pointer");
  HYDRA_REQUIRE(row_stride_bytes >= row_bytes, "rows_take: rows overlap");
  const bool vec = aligned16(x) && row_stride_bytes % 16 == 0 && row_bytes % 16 == 0;
  TakeArgs a{};
  a.x = static_cast<char*>(x);
  a.parents = parents;
  a.row_st = row_stride_bytes;
  a.pieces = vec ? row_bytes / 16 : row_bytes;
  a.N = static_cast<int>(N);
  a.log = 0;
  while ((int64_t(2) << a.log) * N <= kTakeThreads * kTakePieces) ++a.log;
  // narrower ranges where there would be few workgroups, of 64 bytes at least: 16 rows of
  // 8 KB 2.6 us (widest ranges: 5.6), 64 of 32 KB 3.0 (6.0), 256 of 64 KB 6.8 (8.5)
  while (a.log > 2 && (a.pieces >> a.log) < device_cus()) --a.log;
  a.cols = 1 << a.log;
  const int64_t wgs = (a.pieces + a.cols - 1) / a.cols;
  HYDRA_REQUIRE(grid_fits(wgs, kTakeThreads), "rows_take: too large");
  auto st = static_cast<hipStream_t>(stream);
  if (vec) take_rows_kernel<uint4><<<static_cast<unsigned>(wgs), kTakeThreads, 0, st>>>(a);
  else take_rows_kernel<uint8_t><<<static_cast<unsigned>(wgs), kTakeThreads, 0, st>>>(a);
  return check_launch("rows_take");
}
