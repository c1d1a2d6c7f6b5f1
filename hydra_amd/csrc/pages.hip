// Pages of a key-value cache on gfx950: the page tables and slot maps of a
// step from the lengths of its requests, the return of finished requests'
// pages, and the store of key and value rows into their pages.
//
// A cache is a pool of pages, [pages, Hkv, page_size, hd] for keys and for
// values; position t of request i lies in page table[i, t / page_size] at row
// t % page_size, its slot is page * page_size + row.  Pages that nobody holds
// lie on a stack (free_pages[0 .. free_count)).  Nothing here is read by the
// host: a request that cannot get its pages is refused on the device.
#include "common.h"
#include "mod_keys.h"

namespace hydra {
namespace {

constexpr int kPlanThreads = 256;
constexpr int kPlanTokens = 4096;  // tokens of a request that one workgroup writes
constexpr int64_t kMaxPlanned = int64_t(1) << 24;  // requests: each workgroup of a plan goes over those before it

struct PlanArgs {
  const int* lengths;  // may be lengths_out (see hydra_page_plan_in_place)
  const int* fresh;  // tokens to add
  int* table;
  int64_t table_rs;
  const int* free_pages;
  const int* free_count;
  int64_t* slots;
  int* lengths_out;
  int* seen;
  uint8_t* granted;
  int *positions, *free_out;
  int64_t limit;  // tokens of a request at most
  int N, F, width, shift, slice, from_empty;
};

struct Need {
  int64_t len, add;
  int have, need;
  bool fits;
};

// What request i asks for: pages held, pages more, and whether the longest
// request and the step's width allow it.
__device__ __forceinline__ Need need_of(const PlanArgs& a, int i) {
  Need r{0, 0, 0, 0, false};
  if (i >= a.N) return r;
  r.len = a.lengths[i];
  r.add = a.fresh[i];
  const int64_t page = int64_t(1) << a.shift;
  r.fits = r.len >= 0 && r.add >= 0 && r.add <= a.width && r.len + r.add <= a.limit &&
           (!a.from_empty || r.len == 0 || r.add == 0);
  if (r.fits) {
    r.have = static_cast<int>((r.len + page - 1) >> a.shift);
    r.need = static_cast<int>((r.len + r.add + page - 1) >> a.shift) - r.have;
  }
  return r;
}

// Inclusive sum over the workgroup's 256 threads; `total` gets the whole sum.
__device__ __forceinline__ int block_incl_sum(int x, int* part, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int s = wave_incl_sum(x);
  __syncthreads();  // the last use of `part` is over
  if (lane == 63) part[wave] = s;
  __syncthreads();
  int all = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 64; ++w) {
    if (w < wave) s += part[w];
    all += part[w];
  }
  total = all;
  return s;
}

// Workgroup (x, y) writes the results of the requests [x slice, (x+1) slice)
// and, of each, the slots of the tokens [y kPlanTokens, ...).  Every workgroup
// sums the needs of all requests before its own again (256 a step, 8 bytes
// each, from L2): one launch, no exchange between workgroups.  New pages are
// taken from the stack by index, so the table's new entries are written by one
// workgroup and read by none.
//
// Bound by its launch and the chain lengths -> sums -> stack -> slots at a decoding
// step (32 requests: 2.7 us).  For prompts (256 of up to 4096 tokens: 7.0 us, 8 MB
// written at 1.3 TB/s, far below what the memory takes) by the sixteen trips of a
// thread, each a look into the table or the stack for its one token and a store of
// 8 bytes, although the tokens of a page share what is looked up.
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(PlanArgs a) {
  __shared__ int part[kPlanThreads / 64];
  __shared__ int s_first[kPlanThreads], s_have[kPlanThreads], s_need[kPlanThreads];
  __shared__ int64_t s_len[kPlanThreads], s_add[kPlanThreads];  // add: -1 when refused
  const int tid = threadIdx.x;
  const int begin = blockIdx.x * a.slice, end = min(a.N, begin + a.slice);
  int free = *a.free_count;
  free = free < 0 ? 0 : (free > a.F ? a.F : free);
  int before = 0;  // pages asked for by the requests before this step's 256
  int taken = 0;   // pages granted in all (the last workgroup's alone is whole)
  for (int i0 = 0; i0 < end; i0 += kPlanThreads) {
    const int i = i0 + tid;
    const Need r = need_of(a, i);
    int step;
    const int upto = before + block_incl_sum(r.need, part, step);
    const bool granted = r.fits && (r.need == 0 || upto <= free);
    // granted requests that need pages come first, so the last of them
    // has the sum of all
    taken = (granted && r.need > 0) ? upto : taken;
    if (i >= begin && i < end) {
      const int at = i - begin;
      s_first[at] = free - 1 - (upto - r.need);
      s_have[at] = r.have;
      s_need[at] = r.need;
      s_len[at] = r.len;
      s_add[at] = granted ? r.add : -1;
    }
    before += step;
  }
  __syncthreads();
  if (blockIdx.y == 0) {
    for (int at = tid; at < end - begin; at += kPlanThreads) {
      const int i = begin + at;
      const bool granted = s_add[at] >= 0;
      const int after = static_cast<int>(granted ? s_len[at] + s_add[at] : s_len[at]);
      a.lengths_out[i] = after;
      a.seen[i] = granted && s_add[at] > 0 ? after : 0;
      a.granted[i] = granted;
      a.positions[i] = static_cast<int>(s_len[at]);
    }
    // new pages: at most this many a request
    const unsigned most = (a.width >> a.shift) + 2, all = (end - begin) * most;
    for (unsigned e = tid; e < all; e += kPlanThreads) {
      const int at = e / most, j = e - at * most;
      if (s_add[at] >= 0 && j < s_need[at])
        a.table[(begin + at) * a.table_rs + s_have[at] + j] = a.free_pages[s_first[at] - j];
    }
    if (blockIdx.x == gridDim.x - 1) {  // it went over every request
      int most = taken;
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) most = max(most, __shfl_xor(most, off));
      if ((tid & 63) == 0) part[tid >> 6] = most;
      __syncthreads();
      if (tid == 0) {
        for (int w = 1; w < kPlanThreads / 64; ++w) most = max(most, part[w]);
        *a.free_out = free - most;
      }
    }
  }
  const int j0 = blockIdx.y * kPlanTokens, j1 = min(a.width, j0 + kPlanTokens);
  const int64_t low = (int64_t(1) << a.shift) - 1;
  auto slot_of = [&](int at, int j) -> int64_t {
    if (j >= s_add[at]) return -1;
    const int64_t t = s_len[at] + j;
    const int col = static_cast<int>(t >> a.shift);
    const int page = col >= s_have[at] ? a.free_pages[s_first[at] - (col - s_have[at])]
                                       : a.table[(begin + at) * a.table_rs + col];
    return page >= 0 ? (static_cast<int64_t>(page) << a.shift) | (t & low) : -1;
  };
  if (a.slice == 1) {
    int64_t* row = a.slots + static_cast<int64_t>(begin) * a.width;
#pragma unroll 4
    for (int j = j0 + tid; j < j1; j += kPlanThreads) row[j] = slot_of(0, j);
  } else {  // whole rows of several requests, one after the other
    const unsigned width = a.width, count = (end - begin) * width;
    int64_t* rows = a.slots + static_cast<int64_t>(begin) * a.width;
    for (unsigned e = tid; e < count; e += kPlanThreads) {
      const unsigned at = e / width;
      rows[e] = slot_of(at, e - at * width);
    }
  }
}

// The pages of the requests that are done go back on the stack, in the order
// of the requests; their lengths become 0 and their table entries -1.  Entries
// that are no page (outside [0, pages)) do not come back: the next plan would
// hand them to another request.  One workgroup: the stack has one top.  Its
// threads take the entries of 256 requests in their order on the stack, twice
// 256 at once, and look up whose each is; those that are pages are counted only
// where one of them is none.  Bound by the launch and the chain lengths ->
// sums -> table -> stack: 32 of 256 requests with 16 pages each, 3.0 us.
constexpr int kReleaseEntries = 2;

__global__ __launch_bounds__(kPlanThreads) void release_kernel(const uint8_t* done, int* lengths, int* table,
                                                               int64_t table_rs, int* free_pages, int* free_count,
                                                               int N, int P, int F, int pages, int shift) {
  constexpr int U = kReleaseEntries;
  __shared__ int part[kPlanThreads / 64];
  __shared__ int s_upto[kPlanThreads];
  const int tid = threadIdx.x;
  int free = *free_count;
  free = free < 0 ? 0 : (free > F ? F : free);
  for (int i0 = 0; i0 < N; i0 += kPlanThreads) {
    const int i = i0 + tid;
    int count = 0;
    if (i < N && done[i]) {
      const int64_t len = lengths[i];
      const int64_t held = len <= 0 ? 0 : (len + (int64_t(1) << shift) - 1) >> shift;
      count = static_cast<int>(held < P ? held : P);
      lengths[i] = 0;
    }
    int step;
    const int upto = block_incl_sum(count, part, step);
    s_upto[tid] = upto;
    __syncthreads();
    const unsigned entries = step;
    // unsigned: the last trip's indexes, and a full stack's, may pass an int
    for (unsigned e0 = 0; e0 < entries; e0 += kPlanThreads * U) {
      int at[U], page[U];  // at: the first request with s_upto > e
      int* entry[U];
#pragma unroll
      for (int u = 0; u < U; ++u) at[u] = 0;
#pragma unroll
      for (int half = kPlanThreads / 2; half > 0; half >>= 1)
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (static_cast<unsigned>(s_upto[at[u] + half - 1]) <= min(e0 + u * kPlanThreads + tid, entries - 1))
            at[u] += half;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const unsigned e = min(e0 + u * kPlanThreads + tid, entries - 1);
        entry[u] = table + (i0 + at[u]) * table_rs + (e - (at[u] > 0 ? s_upto[at[u] - 1] : 0));
        page[u] = *entry[u];
      }
      bool wrong = false;  // any that is no page
#pragma unroll
      for (int u = 0; u < U; ++u) wrong = wrong || page[u] < 0 || page[u] >= pages;
      const bool all_pages = !__syncthreads_or(wrong);
      unsigned below = free;  // the height of the stack below the next 256
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const unsigned e = e0 + u * kPlanThreads + tid;
        bool back = e < entries;
        if (back) *entry[u] = -1;
        unsigned to = below + tid;
        int more = kPlanThreads;
        if (!all_pages) {
          back = back && page[u] >= 0 && page[u] < pages;
          to = below + block_incl_sum(back, part, more) - 1;
        }
        if (back && to < static_cast<unsigned>(F)) free_pages[to] = page[u];
        below += more;
      }
      if (all_pages) below = min(below, free + (entries - e0));
      free = min(below, static_cast<unsigned>(F));
    }
    __syncthreads();
  }
  if (tid == 0) *free_count = free;
}

// Rows k, v [N, Hkv, S, hd] into their pages.  A thread moves kStorePieces 16-byte
// pieces (elements where rows are not made of such) of key rows and of the value
// rows beside them; neighbouring threads take a row's pieces, then the next
// position's, which lie one after the other in the source and in the page.
// Bound by HBM: each row is read and written once, and not read again soon (so
// past the L2).  64 prompts of up to 4096 tokens, 8 heads of 128, bf16 (262 MB
// moved): 49 us, 5.3 TB/s with three pieces a thread (60 us where the pages lie
// in no order); 3.1 with one, 4.4 with
// two, 4.7 with four (workgroups of 12 KB spread their addresses best).  Fewer
// than 20 MB: 3 to 6 us, the launch.
constexpr int kStorePieces = 3;

struct StoreArgs {
  const char *k, *v;
  char *kp, *vp;
  const int64_t *slots, *rows;  // rows: n -> row of slots (null: n)
  int64_t ks[2], vs[2], kps[2], vps[2];  // strides in bytes: n/h, page/h
  uint32_t k_row, v_row, kp_row, vp_row;
  int64_t limit;                         // slots of the pool
  int N, R, log, shift;                  // log: of pieces, or -1
  uint32_t S, pieces, total;             // total: pieces of a head's rows
};

template <typename V>
__global__ __launch_bounds__(256) void store_kernel(StoreArgs a) {
  constexpr int U = kStorePieces;
  const uint32_t e0 = blockIdx.x * (256 * U) + threadIdx.x;
  const int h = blockIdx.y;
  for (int n = blockIdx.z; n < a.N; n += gridDim.z) {
    const int64_t r = a.rows ? a.rows[n] : n;
    if (r < 0 || r >= a.R) continue;
    const int64_t* slots = a.slots + r * a.S;
    const char *k = a.k + n * a.ks[0] + h * a.ks[1], *v = a.v + n * a.vs[0] + h * a.vs[1];
    int64_t slot[U];
    uint32_t s[U], piece[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t e = min(e0 + 256 * u, a.total - 1);
      s[u] = a.log >= 0 ? e >> a.log : e / a.pieces;
      piece[u] = (e - s[u] * a.pieces) * static_cast<uint32_t>(sizeof(V));
      slot[u] = e0 + 256 * u < a.total ? slots[s[u]] : -1;
    }
    V kv[U], vv[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (slot[u] < 0 || slot[u] >= a.limit) continue;
      kv[u] = *reinterpret_cast<const V*>(k + (static_cast<uint64_t>(s[u]) * a.k_row + piece[u]));
      vv[u] = *reinterpret_cast<const V*>(v + (static_cast<uint64_t>(s[u]) * a.v_row + piece[u]));
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (slot[u] < 0 || slot[u] >= a.limit) continue;
      const int64_t page = slot[u] >> a.shift;
      const uint32_t row = static_cast<uint32_t>(slot[u]) & ((1u << a.shift) - 1);
      char* kp = a.kp + page * a.kps[0] + h * a.kps[1] + (static_cast<uint64_t>(row) * a.kp_row + piece[u]);
      char* vp = a.vp + page * a.vps[0] + h * a.vps[1] + (static_cast<uint64_t>(row) * a.vp_row + piece[u]);
      __builtin_nontemporal_store(kv[u], reinterpret_cast<V*>(kp));
      __builtin_nontemporal_store(vv[u], reinterpret_cast<V*>(vp));
    }
  }
}

// Requests of a workgroup: up to 256, fewer where their slots are many.
int plan_slice(int64_t width) {
  const int64_t slice = kPlanTokens / width;
  return static_cast<int>(slice < 1 ? 1 : (slice > kPlanThreads ? kPlanThreads : slice));
}

int page_shift(int64_t page_size) {
  for (int s = 4; s <= 12; ++s)
    if (page_size == (int64_t(1) << s)) return s;
  return -1;
}

}  // namespace
}  // namespace hydra

using namespace hydra;

extern "C" int hydra_page_plan(const int* lengths, const int* new_tokens, int* table, int64_t table_rs,
                               const int* free_pages, int64_t free_capacity, const int* free_count, int64_t* slots,
                               int* lengths_out, int* seen, void* granted, int* positions, int* free_out,
                               int64_t N, int64_t P, int64_t width, int64_t page_size, int from_empty, void* stream) {
  return hydra_pool_plan(lengths, new_tokens, table, table_rs, free_pages, free_capacity, free_count, slots,
                         lengths_out, seen, granted, positions, free_out, N, P, width, page_size, INT64_MAX, from_empty,
                         stream);
}

extern "C" int hydra_pool_plan(const int* lengths, const int* new_tokens, int* table, int64_t table_rs,
                               const int* free_pages, int64_t free_capacity, const int* free_count, int64_t* slots,
                               int* lengths_out, int* seen, void* granted, int* positions, int* free_out,
                               int64_t N, int64_t P, int64_t width, int64_t page_size, int64_t max_length,
                               int from_empty, void* stream) {
  HYDRA_REQUIRE(N >= 1 && P >= 1 && width >= 1 && free_capacity >= 0 && max_length >= 0, "page_plan: bad size");
  const int shift = page_shift(page_size);
  HYDRA_REQUIRE(shift >= 0, "page_plan: page_size must be a power of two in [16, 4096]");
  HYDRA_REQUIRE(table_rs >= P, "page_plan: table row stride < columns");
  HYDRA_REQUIRE(N <= kMaxPlanned && P < (int64_t(1) << 31) && width < (int64_t(1) << 28) &&
                    N * P < (int64_t(1) << 31) && P * page_size < (int64_t(1) << 31) &&
                    N * width < (int64_t(1) << 40) && free_capacity < (int64_t(1) << 31),
                "page_plan: too large");
  HYDRA_REQUIRE(lengths && new_tokens && table && free_count && slots && lengths_out && seen && granted && positions &&
                    free_out &&
                    (free_pages || free_capacity == 0),
                "page_plan: null pointer");
  HYDRA_REQUIRE((lengths_out != lengths && free_out != free_count) || hydra_page_plan_in_place(N, width) == 1,
                "page_plan: in place takes a step that one workgroup plans");
  PlanArgs a{lengths, new_tokens, table, table_rs, free_pages, free_count, slots, lengths_out, seen,
             static_cast<uint8_t*>(granted), positions, free_out, P * page_size < max_length ? P * page_size : max_length,
             static_cast<int>(N), static_cast<int>(free_capacity), static_cast<int>(width), shift, 0,
             from_empty ? 1 : 0};
  a.slice = plan_slice(width);
  const int64_t gx = (N + a.slice - 1) / a.slice, gy = (width + kPlanTokens - 1) / kPlanTokens;
  HYDRA_REQUIRE(gx < (int64_t(1) << 31) && gy <= 65535, "page_plan: too large");
  plan_kernel<<<dim3(static_cast<unsigned>(gx), static_cast<unsigned>(gy)), kPlanThreads, 0,
                static_cast<hipStream_t>(stream)>>>(a);
  return check_launch("page_plan");
}

// A lone workgroup has read every length, and the stack's height, before it
// writes its first result.
extern "C" int hydra_page_plan_in_place(int64_t N, int64_t width) {
  return N >= 1 && width >= 1 && width <= kPlanTokens && N <= plan_slice(width) ? 1 : 0;
}

extern "C" int hydra_page_release(const void* done, int* lengths, int* table, int64_t table_rs, int* free_pages,
                                  int64_t free_capacity, int* free_count, int64_t N, int64_t P, int64_t page_size,
                                  void* stream) {
  return hydra_pool_release(done, lengths, table, table_rs, free_pages, free_capacity, free_count, N, P, page_size,
                            INT32_MAX, stream);
}

extern "C" int hydra_pool_release(const void* done, int* lengths, int* table, int64_t table_rs, int* free_pages,
                                  int64_t free_capacity, int* free_count, int64_t N, int64_t P, int64_t page_size,
                                  int64_t pages, void* stream) {
  HYDRA_REQUIRE(N >= 1 && P >= 1 && free_capacity >= 1 && pages >= 1, "page_release: bad size");
  const int shift = page_shift(page_size);
  HYDRA_REQUIRE(shift >= 0, "page_release: page_size must be a power of two in [16, 4096]");
  HYDRA_REQUIRE(table_rs >= P, "page_release: table row stride < columns");
  HYDRA_REQUIRE(N <= kMaxPlanned && P < (int64_t(1) << 31) && N * P < (int64_t(1) << 31) &&
                    free_capacity < (int64_t(1) << 31) && pages < (int64_t(1) << 31),
                "page_release: too large");
  HYDRA_REQUIRE(done && lengths && table && free_pages && free_count, "page_release: null pointer");
  release_kernel<<<1, kPlanThreads, 0, static_cast<hipStream_t>(stream)>>>(
      static_cast<const uint8_t*>(done), lengths, table, table_rs, free_pages, free_count, static_cast<int>(N),
      static_cast<int>(P), static_cast<int>(free_capacity), static_cast<int>(pages), shift);
  return check_launch("page_release");
}

extern "C" int hydra_page_store(const void* k, const void* v, void* k_pages, void* v_pages, const int64_t* slots,
                                int64_t R, const int64_t* rows, int64_t N, int64_t Hkv, int64_t S, int64_t hd,
                                int64_t pages, int64_t page_size, const int64_t* k_st, const int64_t* v_st,
                                const int64_t* kp_st, const int64_t* vp_st, int dtype, void* stream) {
  HYDRA_REQUIRE(N >= 0 && S >= 0 && R >= 0 && Hkv >= 1 && hd >= 1 && pages >= 1, "page_store: bad size");
  HYDRA_REQUIRE(rows || R >= N, "page_store: fewer rows of slots than prompts");
  const int shift = page_shift(page_size);
  HYDRA_REQUIRE(shift >= 0, "page_store: page_size must be a power of two in [16, 4096]");
  const int e = dtype_size(dtype);
  HYDRA_REQUIRE(e > 0, "page_store: unknown dtype");
  HYDRA_REQUIRE(N < (int64_t(1) << 31) && R < (int64_t(1) << 31) && S < (int64_t(1) << 31) && Hkv <= 65535 &&
                    hd <= 65536 && pages < (int64_t(1) << 31),
                "page_store: too large");
  if (N == 0 || S == 0) return HYDRA_OK;
  HYDRA_REQUIRE(k && v && k_pages && v_pages && slots && k_st && v_st && kp_st && vp_st, "page_store: null pointer");
  HYDRA_REQUIRE(k_st[3] == 1 && v_st[3] == 1 && kp_st[3] == 1 && vp_st[3] == 1, "page_store: rows need unit stride");
  StoreArgs a{};
  a.k = static_cast<const char*>(k);
  a.v = static_cast<const char*>(v);
  a.kp = static_cast<char*>(k_pages);
  a.vp = static_cast<char*>(v_pages);
  a.slots = slots;
  a.rows = rows;
  a.R = static_cast<int>(R);
  a.limit = pages * page_size;
  a.N = static_cast<int>(N);
  a.S = static_cast<uint32_t>(S);
  a.shift = shift;
  bool vec = hd * e % 16 == 0 && aligned16(k) && aligned16(v) && aligned16(k_pages) && aligned16(v_pages);
  for (int i = 0; i < 2; ++i) {
    a.ks[i] = k_st[i] * e;
    a.vs[i] = v_st[i] * e;
    a.kps[i] = kp_st[i] * e;
    a.vps[i] = vp_st[i] * e;
    vec = vec && (a.ks[i] | a.vs[i] | a.kps[i] | a.vps[i]) % 16 == 0;
  }
  uint32_t* const row[4] = {&a.k_row, &a.v_row, &a.kp_row, &a.vp_row};
  for (int i = 0; i < 4; ++i) {
    const int64_t st = (i == 0 ? k_st : i == 1 ? v_st : i == 2 ? kp_st : vp_st)[2] * e;
    HYDRA_REQUIRE(st >= 0 && st < (int64_t(1) << 32), "page_store: rows too far apart");
    *row[i] = static_cast<uint32_t>(st);
    vec = vec && st % 16 == 0;
  }
  a.pieces = static_cast<uint32_t>(vec ? hd * e / 16 : hd);
  a.log = (a.pieces & (a.pieces - 1)) == 0 ? __builtin_ctz(a.pieces) : -1;
  HYDRA_REQUIRE(S * a.pieces < (int64_t(1) << 31), "page_store: too large");
  a.total = a.S * a.pieces;
  const int64_t z = N < 65535 ? N : 65535;
  const unsigned span = 256 * kStorePieces;
  const dim3 grid((a.total + span - 1) / span, static_cast<unsigned>(Hkv), static_cast<unsigned>(z));
  auto st = static_cast<hipStream_t>(stream);
  if (vec) store_kernel<u32x4_nt><<<grid, 256, 0, st>>>(a);
  else if (e == 4) store_kernel<uint32_t><<<grid, 256, 0, st>>>(a);
  else store_kernel<uint16_t><<<grid, 256, 0, st>>>(a);
  return check_launch("page_store");
}
