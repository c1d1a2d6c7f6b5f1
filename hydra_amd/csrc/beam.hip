// A step of beam search on gfx950: of each text's W beams the best n
// continuations,
//
//   top n over (w, v) of  score[w] + x[w, v] - ln sum_u e^(x[w, u]),
//
// in descending order, the lowest w V + v first among equals.
//
// Bound by one pass over the logits where texts are many: 32 texts of 8 beams by 32000,
// bf16 (16 MB), n = 16: 10.4 us, and 8.3 to join; for one text of 4 beams by 50257, n = 4,
// by latency: 5.7 and 5.8 us.  Each workgroup reads a chunk of a row into
// registers, takes its maximum and its sum of exponentials (fp32) and leaves the
// chunk's n best (value, index) pairs; a second kernel joins the chunks' sums,
// and orders the chunks' pairs by their scores in fp64 (two beams' continuations may be
// closer than fp32 tells).  Within a row the order is that of the logits
// themselves.
//
// The n best of a workgroup's elements, without sorting them: the threads fall
// into four n groups or so, and the n-th largest of the groups' maxima is a bound that
// n elements reach; those that do (a few more than n, whatever the order of the
// elements) are collected and ranked by counting.  Keys are unique (an index is part of
// them), so the order in which they are collected does not matter.
//
// Chunks that the join reads again, since fp64 tells none of their logits apart, cost it far
// more: 614 us with all beams of the 32 texts at a score of -1e30, 114 with all logits 0.
#include "common.h"
#include "mod_keys.h"

namespace hydra {
namespace {

constexpr int kThreads = 256;
constexpr int kCap = 2048;       // collected elements
constexpr int kFew = 64;         // elements that are ranked as they are, which takes a comparison for each thread
constexpr int kMaxCount = 128;   // n
constexpr int kMaxBeams = 1024;  // W

// Larger is better; 0 is none.  Of a chunk: the value's key and ~index; of a text:
// the score's key, and ~(w V + v) beside it.
struct Key1 {
  uint64_t a;
};
struct Key2 {
  uint64_t a;
  uint32_t b;
};
__device__ __forceinline__ bool better(const Key1& x, const Key1& y) { return x.a > y.a; }
__device__ __forceinline__ bool better(const Key2& x, const Key2& y) { return x.a > y.a || (x.a == y.a && x.b > y.b); }
// In the keys' order, equal ones in any.
template <typename Key>
__device__ __forceinline__ uint32_t rough(const Key& k) {
  return static_cast<uint32_t>(k.a >> 32);
}

template <typename Key> struct Lists {
  Key list[kCap];
  alignas(16) uint32_t part[kThreads];
  Key nth;
  uint32_t bound;
  int count;
};

// A bound that n threads' `mine` reach, and few more (all 256 take part).
template <typename Key>
__device__ __forceinline__ uint32_t bound_of(uint32_t mine, int n, Lists<Key>& L) {
  int size = 64;  // threads of a group
  while (size > 1 && kThreads / size < 4 * n) size >>= 1;
  for (int o = 1; o < size; o <<= 1) mine = max(mine, static_cast<uint32_t>(__shfl_xor(static_cast<int>(mine), o)));
  const int groups = kThreads / size;
  if (threadIdx.x % size == 0) L.part[threadIdx.x / size] = mine;
  if (threadIdx.x == 0) L.bound = 0xffffffffu;
  __syncthreads();
  if (threadIdx.x < groups) {
    const uint4* part = reinterpret_cast<const uint4*>(L.part);
    mine = L.part[threadIdx.x];
    int above = 0;
    for (int i = 0; i < groups / 4; ++i) {
      const uint4 p = part[i];
      above += (p.x > mine) + (p.y > mine) + (p.z > mine) + (p.w > mine);
    }
    if (above < n) atomicMin(&L.bound, mine);
  }
  __syncthreads();
  return L.bound;
}

// A place in the list for each lane with `in`: one count for the wave.
__device__ __forceinline__ int place(bool in, int* count) {
  const uint64_t who = __ballot(in);
  if (who == 0) return 0;
  int base = 0;
  if ((threadIdx.x & 63) == __ffsll(static_cast<unsigned long long>(who)) - 1) base = atomicAdd(count, __popcll(who));
  base = __shfl(base, __ffsll(static_cast<unsigned long long>(who)) - 1);
  return base + __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(who >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(who), 0));
}

// The list's c elements by ranks, to put(rank, key), as far as the ranks are below n.
template <typename Key, typename Put>
__device__ __forceinline__ void counted(int n, int c, Lists<Key>& L, Put&& put) {
  // four lanes to an element, a quarter of the list each
  const int tid = threadIdx.x, q = tid & 3, i0 = c * q / 4, i1 = c * (q + 1) / 4;
  for (int j0 = 0; j0 < c; j0 += kThreads / 4) {
    const int j = j0 + (tid >> 2);
    const Key k = L.list[min(j, c - 1)];
    int rank = 0;
#pragma unroll 4
    for (int i = i0; i < i1; ++i) rank += better(L.list[i], k);
    rank += __shfl_xor(rank, 1);
    rank += __shfl_xor(rank, 2);
    if (q == 0 && j < c && k.a != 0 && rank < n) put(rank, k);
  }
}

// The n best of the list's c elements, best first, to put(rank, key); ranks without an
// element get none.
template <typename Key, typename Put>
__device__ __forceinline__ void ranked(int n, int c, Lists<Key>& L, Put&& put) {
  constexpr int U = kCap / kThreads;
  const int tid = threadIdx.x;
  // many: those that reach a bound of the list's own elements move to its front
  for (int i = 0; i < 2 && c > 128 && c > 2 * n; ++i) {
    Key mine[U];
    uint32_t top = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      mine[u] = Key{};
      if (u * kThreads + tid < c) mine[u] = L.list[u * kThreads + tid];
      top = max(top, rough(mine[u]));
    }
    const uint32_t bound = bound_of(top, n, L);  // everybody has read
    if (tid == 0) L.count = 0;
    __syncthreads();
    const int trips = (c + kThreads - 1) / kThreads;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u >= trips) continue;
      const bool in = mine[u].a != 0 && rough(mine[u]) >= bound;
      const int at = place(in, &L.count);
      if (in) L.list[at] = mine[u];
    }
    __syncthreads();
    c = L.count;
    __syncthreads();
  }
  counted(n, c, L, put);
  for (int j = c + tid; j < n; j += kThreads) put(j, Key{});
}

// At least the n best of all elements into the list; their number.  Any n elements give a
// bound: first the threads' best ones, then those of a list that was too short.
template <typename Key, typename Each>
__device__ __forceinline__ int collected(int n, Lists<Key>& L, Each&& each) {
  Key best{};
  each([&](const Key& k) {
    if (better(k, best)) best = k;
  });
  __syncthreads();
  L.list[threadIdx.x] = best;
  for (int c = kThreads;; c = kCap) {
    if (threadIdx.x == 0) {
      L.nth = Key{};
      L.count = 0;
    }
    __syncthreads();
    counted(n, c, L, [&](int rank, const Key& k) {
      if (rank == n - 1) L.nth = k;
    });
    __syncthreads();
    const Key nth = L.nth;
    each([&](const Key& k) {
      if (k.a == 0 || better(nth, k)) return;
      const int at = atomicAdd(&L.count, 1);
      if (at < kCap) L.list[at] = k;
    });
    __syncthreads();
    const int count = L.count;
    if (count <= kCap) return count;
    __syncthreads();
  }
}

// A chunk's results: maximum, sum of e^(x - maximum), and pairs (key of the value, ~index).
struct BeamArgs {
  const char* logits;
  const float* scores;
  float* stats;       // [rows][chunks][2]
  uint2* pairs;       // [rows][chunks][n]
  float* out_scores;
  int64_t *beams, *tokens;
  int* parents;
  int64_t stride;     // bytes of a row
  int B, W, V, n, chunks;
  int span;           // elements of a chunk
  int first;          // row (text) of the launch's first workgroup
};

__device__ __forceinline__ Key1 key_of(float v, int i) {
  return Key1{(static_cast<uint64_t>(score_key_asc(v)) << 32) | (0xffffffffu - static_cast<uint32_t>(i))};
}

__device__ __forceinline__ float key_float(uint32_t k) {
  return __uint_as_float(k >> 31 ? k & 0x7fffffffu : ~k);
}

template <typename T, int E>
__global__ __launch_bounds__(kThreads) void beam_chunk_kernel(BeamArgs a) {
  constexpr int N = Vec<T>::N, J = E / N;
  __shared__ Lists<Key1> lists;
  __shared__ float red[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = a.first + blockIdx.y, c0 = blockIdx.x * (E * kThreads);
  const T* x = reinterpret_cast<const T*>(a.logits + row * a.stride);
  // the row's elements before the first 16-byte boundary count as chunk 0's first piece
  const int off = static_cast<int>(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T));
  float v[E];
  float top = -INFINITY;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int i = c0 + (j * kThreads + tid) * N - off;  // index of the piece's first element
    if (i >= 0 && i + N <= a.V) {
      load16<T, true>(x + i, v + j * N);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) v[j * N + e] = i + e >= 0 && i + e < a.V ? to_f32(x[i + e]) : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < N; ++e) top = fmaxf(top, v[j * N + e]);
  }
  const uint32_t mine = score_key_asc(top);
  top = wave_max(top);
  if (lane == 0) red[wave] = top;
  __syncthreads();
  top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float ts = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < E; ++j) sum += __expf(v[j] - ts);  // elements that are none: e^-inf
  sum = wave_sum(sum);
  __syncthreads();
  if (lane == 0) red[wave] = sum;
  __syncthreads();
  const int64_t at = static_cast<int64_t>(row) * a.chunks + blockIdx.x;
  if (tid == 0) {
    a.stats[2 * at] = top;
    a.stats[2 * at + 1] = red[0] + red[1] + red[2] + red[3];
  }
  auto each = [&](auto&& f) {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int i = c0 + (j * kThreads + tid) * N - off;
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (i + e >= 0 && i + e < a.V) f(key_of(v[j * N + e], i + e));
    }
  };
  uint2* out = a.pairs + at * a.n;
  auto put = [&](int rank, const Key1& k) {
    out[rank] = make_uint2(static_cast<uint32_t>(k.a >> 32), static_cast<uint32_t>(k.a));
  };
  // By the values alone first, which is a comparison for each element.  (A NaN is below
  // everything here: its row counts as NaN throughout.)
  const float bound = key_float(bound_of(mine, a.n, lists));
  if (tid == 0) lists.count = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int i = c0 + (j * kThreads + tid) * N - off;
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (v[j * N + e] >= bound) {  // few; what lies outside the row is -inf
        if (i + e >= 0 && i + e < a.V) {
          const int to = atomicAdd(&lists.count, 1);
          if (to < kCap) lists.list[to] = key_of(v[j * N + e], i + e);
        }
      }
  }
  __syncthreads();
  int c = lists.count;
  if (c > kCap) c = collected(a.n, lists, each);  // many equal ones (masked rows): by value and index
  ranked(a.n, c, lists, put);
}

__device__ __forceinline__ uint64_t double_key(double v) {  // ascending; NaN above all, -0 as 0
  if (v != v) return ~0ull;
  const uint64_t u = static_cast<uint64_t>(__double_as_longlong(v == 0.0 ? 0.0 : v));
  return u >> 63 ? ~u : u | (1ull << 63);
}
__device__ __forceinline__ double key_double(uint64_t k) {
  if (k == ~0ull) return __longlong_as_double(0x7ff8000000000000ll);
  return __longlong_as_double(static_cast<long long>(k >> 63 ? k & ~(1ull << 63) : ~k));
}

template <typename T>
__global__ __launch_bounds__(kThreads) void beam_join_kernel(BeamArgs a) {
  __shared__ Lists<Key2> lists;
  // x - top first: a row whose tokens are all masked by the type's lowest value is even
  __shared__ double shift[kMaxBeams];  // score - ln sum e^(x - top)
  __shared__ float tops[kMaxBeams];
  __shared__ int cut;  // whether a list may end among equals
  const int tid = threadIdx.x, b = a.first + blockIdx.x;
  const int count = a.W * a.chunks, all = count * a.n;  // lists, and what they hold
  const uint2* pairs = a.pairs + static_cast<int64_t>(b) * all;
  // The lists by ranks: all lists' best, then all lists' second, so that neighbours, which
  // are in different groups, are much alike.  A thread's first ones are under way while the
  // sums are joined.
  auto pair_at = [&](int i) {
    const int rank = i / count;
    return pairs[static_cast<int64_t>(i - rank * count) * a.n + rank];
  };
  constexpr int U = 4;
  uint2 early[U];
#pragma unroll
  for (int u = 0; u < U; ++u) early[u] = u * kThreads + tid < all ? pair_at(u * kThreads + tid) : make_uint2(0, 0);
  if (tid == 0) cut = 0;
  // where a list ends, for the threads' first ones
  auto last_of = [&](int l) { return pairs[static_cast<int64_t>(l) * a.n + a.n - 1]; };
  const uint32_t early_last = tid < count ? last_of(tid).x : 0;
  // as many lanes to a row as it has chunks
  int lanes = 1;
  while (lanes < 64 && lanes < a.chunks) lanes *= 2;
  const int sub = tid & (lanes - 1);
  for (int w0 = 0; w0 < a.W; w0 += kThreads / lanes) {
    const int w = min(w0 + tid / lanes, a.W - 1);
    const float2* st = reinterpret_cast<const float2*>(a.stats) + (static_cast<int64_t>(b) * a.W + w) * a.chunks;
    float top = -INFINITY;
    for (int c = sub; c < a.chunks; c += lanes) top = fmaxf(top, st[c].x);
    for (int o = 1; o < lanes; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
    const double ts = top == -INFINITY ? 0.0 : top;
    double sum = 0.0;
    for (int c = sub; c < a.chunks; c += lanes) {
      const float2 s = st[c];
      sum += s.x == -INFINITY && s.y == 0.f ? 0.0 : s.y * exp(s.x - ts);
    }
    for (int o = 1; o < lanes; o <<= 1) sum += __shfl_xor(sum, o);
    if (sub == 0) {  // a row of -inf alone has log probabilities -inf
      shift[w] = sum == 0.0 && top == -INFINITY ? -INFINITY : a.scores[static_cast<int64_t>(b) * a.W + w] - log(sum);
      tops[w] = static_cast<float>(ts);
    }
  }
  __syncthreads();
  auto key_of_score = [&](int w, uint32_t value) {  // of a beam whose shift is finite
    return double_key(static_cast<double>(key_float(value)) - static_cast<double>(tops[w]) + shift[w]);
  };
  auto key_at = [&](int i, uint2 p) {
    const int rank = i / count, x = i - rank * count, w = x / a.chunks;
    const double s = shift[w];
    if (!(fabs(s) < INFINITY))  // all of the beam's continuations are equal: its first ones
      return x == w * a.chunks && rank < a.V ? Key2{double_key(s), 0xffffffffu - static_cast<uint32_t>(w * a.V + rank)}
                                             : Key2{0, 0};
    if (p.x == 0) return Key2{0, 0};
    return Key2{key_of_score(w, p.x), 0xffffffffu - static_cast<uint32_t>(w * a.V + static_cast<int>(0xffffffffu - p.y))};
  };
  auto each = [&](auto&& f) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (u * kThreads + tid < all) f(key_at(u * kThreads + tid, early[u]));
    for (int i = U * kThreads + tid; i < all; i += kThreads) f(key_at(i, pair_at(i)));
  };
  auto put = [&](int rank, const Key2& k) {
    const int flat = static_cast<int>(0xffffffffu - k.b), w = flat / a.V;
    const int64_t at = static_cast<int64_t>(b) * a.n + rank;
    a.out_scores[at] = static_cast<float>(key_double(k.a));
    a.beams[at] = w;
    a.tokens[at] = flat - w * a.V;
    a.parents[at] = b * a.W + w;
    if (rank == a.n - 1) lists.nth = k;
  };
  // A list has its chunk's best logits.  Where fp64 does not tell the scores of different
  // logits apart (a beam's score of -1e30, logits of 1e-30) they are equal, and the lowest
  // tokens come first, which a list may have left out.
  auto alike = [&](int l, uint32_t x) {  // x: the key of its last logit
    const int w = l / a.chunks;
    const float v = fabsf(key_float(x)), s = fabsf(static_cast<float>(shift[w]));
    // the next logits are at 2^-25 v at least, a score's two roundings 2^-51 of its terms: most
    // lists end here
    if (v * 0x1p20f > v + fabsf(tops[w]) + s) return false;
    const uint64_t k = key_of_score(w, x);
    return fabs(shift[w]) < INFINITY && x > score_key_asc(-INFINITY) &&
           (key_of_score(w, x - 1) == k || key_of_score(w, x + 1) == k);
  };
  if (tid < count && alike(tid, early_last)) cut = 1;
  for (int l = kThreads + tid; l < count; l += kThreads)
    if (alike(l, last_of(l).x)) cut = 1;
  int c = all;
  if (all <= kFew) {
    if (tid < all) lists.list[tid] = key_at(tid, early[0]);
    __syncthreads();
  } else {
    uint32_t mine = 0;
    each([&](const Key2& k) { mine = max(mine, rough(k)); });
    const uint32_t bound = bound_of(mine, a.n, lists);
    if (tid == 0) lists.count = 0;
    __syncthreads();
    each([&](const Key2& k) {
      if (k.a == 0 || rough(k) < bound) return;
      const int at = atomicAdd(&lists.count, 1);
      if (at < kCap) lists.list[at] = k;
    });
    __syncthreads();
    c = lists.count;
    if (c > kCap) c = collected(a.n, lists, each);
  }
  ranked(a.n, c, lists, put);
  if (cut == 0) return;
  // Chunks whose list's last score is the n-th, and that of a logit beside it, are read again.
  __syncthreads();
  const uint64_t nth = lists.nth.a;
  auto is_cut = [&](int l, uint32_t x) { return alike(l, x) && key_of_score(l / a.chunks, x) == nth; };
  int some = 0;
  for (int l = tid; l < count; l += kThreads) some |= is_cut(l, last_of(l).x);
  if (!__syncthreads_or(some)) return;
  auto with_chunks = [&](auto&& f) {
    each(f);
    for (int l = 0; l < count; ++l) {
      const uint2 last = last_of(l);
      if (!is_cut(l, last.x)) continue;
      const int w = l / a.chunks;
      const Key1 listed{(static_cast<uint64_t>(last.x) << 32) | last.y};  // as far as the list goes
      const T* x = reinterpret_cast<const T*>(a.logits + (static_cast<int64_t>(b) * a.W + w) * a.stride);
      const int c0 = (l - w * a.chunks) * a.span - static_cast<int>(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T));
      for (int i = max(c0, 0) + tid; i < min(c0 + a.span, a.V); i += kThreads) {
        const Key1 k = key_of(to_f32(x[i]), i);
        if (better(listed, k))
          f(Key2{key_of_score(w, static_cast<uint32_t>(k.a >> 32)), 0xffffffffu - static_cast<uint32_t>(w * a.V + i)});
      }
    }
  };
  ranked(a.n, collected(a.n, lists, with_chunks), lists, put);
}

// Elements of a thread.  Longer chunks leave less to join: in a graph, 16 against 32, us,
//   n = 1, 1 beam by 50257: 8.4 : 9.2        n = 4, 4 beams by 50257: 10.6 : 11.5
//   n = 4, 32 x 8 by 32000: 13.4 : 13.5      n = 16, 4 x 8 by 32000: 15.3 : 14.2
//   n = 16, 16 by 32000: 17.6 : 15.6         n = 32, 32 x 16 by 50257: 60 : 49
// and 8 lost to 16 throughout (n = 4, 4 beams by 50257: equal; n = 16, 16 by 32000: 27 : 21).
int elements_of(int64_t n) { return n <= 8 ? 16 : 32; }

// A row that begins inside 16 bytes reaches up to 7 elements further.
int64_t chunks_of(int64_t V, int64_t n) {
  const int64_t c = static_cast<int64_t>(elements_of(n)) * kThreads;
  return (V + 7 + c - 1) / c;
}

int check_beam(int64_t B, int64_t W, int64_t V, int64_t n, int dtype) {
  HYDRA_REQUIRE(B >= 0 && W >= 1 && V >= 1 && n >= 1, "beam_select: bad size");
  HYDRA_REQUIRE(V <= (int64_t(1) << 31) - (1 << 14), "beam_select: vocabulary must be at most 2^31 - 2^14");  // a chunk's end in 32 bits
  HYDRA_REQUIRE(W <= kMaxBeams && n <= kMaxCount, "beam_select: at most 1024 beams and 128 continuations of a text");
  HYDRA_REQUIRE(W * V < (int64_t(1) << 31) && n <= W * V,
                "beam_select: continuations must be at most beams x vocabulary, and these below 2^31");
  HYDRA_REQUIRE(dtype_size(dtype) > 0, "beam_select: unknown dtype");
  HYDRA_REQUIRE(B < (int64_t(1) << 31) / W, "beam_select: too large");
  return HYDRA_OK;
}

int64_t stats_bytes(int64_t rows, int64_t chunks) { return (rows * chunks * 8 + 15) / 16 * 16; }

template <typename T>
int launch_beam(BeamArgs a, int e, hipStream_t st) {
  const int64_t rows = static_cast<int64_t>(a.B) * a.W;
  for (int64_t r = 0; r < rows; r += 65535) {
    a.first = static_cast<int>(r);
    const dim3 grid(static_cast<unsigned>(a.chunks), static_cast<unsigned>(rows - r < 65535 ? rows - r : 65535));
    if (e == 32) beam_chunk_kernel<T, 32><<<grid, kThreads, 0, st>>>(a);
    else beam_chunk_kernel<T, 16><<<grid, kThreads, 0, st>>>(a);
  }
  constexpr int64_t most = int64_t(1) << 22;  // HIP counts a launch's threads in 32 bits
  for (int64_t b = 0; b < a.B; b += most) {
    a.first = static_cast<int>(b);
    beam_join_kernel<T><<<static_cast<unsigned>(a.B - b < most ? a.B - b : most), kThreads, 0, st>>>(a);
  }
  return check_launch("beam_select");
}

}  // namespace
}  // namespace hydra

using namespace hydra;

extern "C" int hydra_beam_select_workspace(int64_t B, int64_t W, int64_t V, int64_t n, int dtype, int64_t* bytes) {
  const int rc = check_beam(B, W, V, n, dtype);
  if (rc != HYDRA_OK) return rc;
  HYDRA_REQUIRE(bytes != nullptr, "beam_select_workspace: null pointer");
  const int64_t rows = B * W, chunks = B == 0 ? 0 : chunks_of(V, n);
  *bytes = stats_bytes(rows, chunks) + rows * chunks * n * 8;
  return HYDRA_OK;
}

extern "C" int hydra_beam_select(const void* logits, int64_t logits_rs, const float* scores, int64_t B, int64_t W,
                                 int64_t V, int64_t n, float* out_scores, int64_t* beams, int64_t* tokens, int* parents,
                                 int dtype, void* workspace, int64_t workspace_size, void* stream) {
  const int rc = check_beam(B, W, V, n, dtype);
  if (rc != HYDRA_OK) return rc;
  if (B == 0) return HYDRA_OK;
  HYDRA_REQUIRE(logits && scores && out_scores && beams && tokens && parents, "beam_select: null pointer");
  HYDRA_REQUIRE(logits_rs >= V || B * W == 1, "beam_select: row stride < vocabulary");
  HYDRA_REQUIRE(reinterpret_cast<uintptr_t>(logits) % dtype_size(dtype) == 0, "beam_select: logits are not aligned to their type");
  const int64_t rows = B * W, chunks = chunks_of(V, n);
  HYDRA_REQUIRE(workspace && aligned16(workspace) && workspace_size >= stats_bytes(rows, chunks) + rows * chunks * n * 8,
                "beam_select: workspace too small");
  BeamArgs a{};
  a.logits = static_cast<const char*>(logits);
  a.scores = scores;
  a.stats = static_cast<float*>(workspace);
  a.pairs = reinterpret_cast<uint2*>(static_cast<char*>(workspace) + stats_bytes(rows, chunks));
  a.out_scores = out_scores;
  a.beams = beams;
  a.tokens = tokens;
  a.parents = parents;
  a.stride = logits_rs * dtype_size(dtype);
  a.B = static_cast<int>(B);
  a.W = static_cast<int>(W);
  a.V = static_cast<int>(V);
  a.n = static_cast<int>(n);
  a.chunks = static_cast<int>(chunks);
  a.span = elements_of(n) * kThreads;
  auto st = static_cast<hipStream_t>(stream);
  return HYDRA_DISPATCH_DTYPE(dtype, T, [&]() -> int { return launch_beam<T>(a, elements_of(n), st); });
}
