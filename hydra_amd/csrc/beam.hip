// A step of beam search on gfx950: of each text's W beams the best n
// continuations,
//
//   top n over (w, v) of  score[w] + x[w, v] - ln sum_u e^(x[w, u]),
//
// in descending order, the lowest w V + v first among equals.
//
// Bound by one pass over the logits.  Each workgroup reads a chunk of a row into
// registers, takes its maximum and its sum of exponentials (fp32) and leaves the
// chunk's n best (value, index) pairs; a second kernel joins the chunks' sums,
// and orders the chunks' pairs by their scores in fp64 (two beams' continuations may be
// closer than fp32 tells).  Within a row the order is that of the logits
// themselves.
//
// The n best of a workgroup's elements, without sorting them: the threads fall
// into at least n groups, and the least of the groups' maxima is a bound that n
// elements reach; those that do (of 4000 even ones, and n = 16, some 50) are
// collected and ranked by counting.  Keys are unique (an index is part of them),
// so the order in which they are collected does not matter.
#include "common.h"
#include "mod_keys.h"

namespace hydra {
namespace {

constexpr int kThreads = 256;
constexpr int kCap = 2048;       // collected elements
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
__device__ __forceinline__ Key1 shuffled(const Key1& k, int off) {
  return Key1{static_cast<uint64_t>(__shfl_xor(static_cast<long long>(k.a), off))};
}
__device__ __forceinline__ Key2 shuffled(const Key2& k, int off) {
  return Key2{static_cast<uint64_t>(__shfl_xor(static_cast<long long>(k.a), off)),
              static_cast<uint32_t>(__shfl_xor(static_cast<int>(k.b), off))};
}

template <typename Key> struct Lists {
  Key list[kCap];
  Key part[kThreads];
  int count;
};

// The least of the maxima of n' >= n groups of threads (all 256 take part): at
// least n elements reach it, if there are as many as groups.  Thread t is in group t mod
// n': neighbours hold neighbouring elements, of one beam or one end of a row, and groups
// of such would be of very different size.
template <typename Key>
__device__ __forceinline__ Key bound_of(Key mine, int n, Key* part) {
  int groups = 1;
  while (groups < n) groups <<= 1;
  const int tid = threadIdx.x, lane = tid & 63;
  for (int off = 32; off >= groups; off >>= 1) {
    const Key o = shuffled(mine, off);
    if (better(o, mine)) mine = o;
  }
  __syncthreads();  // the last use of `part` is over
  part[tid] = mine;
  __syncthreads();
  const int step = groups < 64 ? 64 : groups;  // threads of one group in other waves
  for (int o = (tid + step) & (kThreads - 1); o != tid; o = (o + step) & (kThreads - 1))
    if (better(part[o], mine)) mine = part[o];
  for (int off = 1; off < groups && off < 64; off <<= 1) {
    const Key o = shuffled(mine, off);
    if (better(mine, o)) mine = o;
  }
  if (groups > 64) {  // 128: two waves' groups
    __syncthreads();
    if (lane == 0) part[tid >> 6] = mine;
    __syncthreads();
    if (better(mine, part[(tid >> 6) ^ 1])) mine = part[(tid >> 6) ^ 1];
  }
  return mine;
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

// The n best of the list's c elements, best first, to put(rank, key); ranks without an
// element get none.
template <typename Key, typename Put>
__device__ __forceinline__ void ranked(int n, int c, Lists<Key>& L, Put&& put) {
  constexpr int U = kCap / kThreads;
  const int tid = threadIdx.x;
  // many: those that reach a bound of the list's own elements move to its front
  for (int i = 0; i < 4 && c > 128 && c > 2 * n; ++i) {
    Key mine[U], k{};
#pragma unroll
    for (int u = 0; u < U; ++u) {
      mine[u] = Key{};
      if (u * kThreads + tid < c) mine[u] = L.list[u * kThreads + tid];
      if (better(mine[u], k)) k = mine[u];
    }
    if (tid == 0) L.count = 0;
    const Key tight = bound_of(k, n, L.part);  // everybody has read
    const int trips = (c + kThreads - 1) / kThreads;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u >= trips) continue;
      const bool in = mine[u].a != 0 && !better(tight, mine[u]);
      const int at = place(in, &L.count);
      if (in) L.list[at] = mine[u];
    }
    __syncthreads();
    c = L.count;
    __syncthreads();
  }
  // four lanes to an element, a quarter of the list each
  const int q = tid & 3, i0 = c * q / 4, i1 = c * (q + 1) / 4;
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
  for (int j = c + tid; j < n; j += kThreads) put(j, Key{});
}

// The n best of the elements that each thread's `each` goes over, one after the other: the
// best below the last.
template <typename Key, typename Each, typename Put>
__device__ __forceinline__ void one_by_one(int n, Lists<Key>& L, Each&& each, Put&& put) {
  Key last{};
  for (int i = 0; i < n; ++i) {
    Key k{};
    each([&](const Key& x) {
      if ((i == 0 || better(last, x)) && better(x, k)) k = x;
    });
    for (int off = 1; off < 64; off <<= 1) {
      const Key o = shuffled(k, off);
      if (better(o, k)) k = o;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) L.part[threadIdx.x >> 6] = k;
    __syncthreads();
    for (int w = 0; w < kThreads / 64; ++w)
      if (better(L.part[w], k)) k = L.part[w];
    if (threadIdx.x == 0) put(i, k);
    last = k;
  }
}

// Those of all elements that reach `bound`, which at least n do, into the list; their
// number, which may be more than the list holds.
template <typename Key, typename Each>
__device__ __forceinline__ int collected(const Key& bound, Lists<Key>& L, Each&& each) {
  if (threadIdx.x == 0) L.count = 0;
  __syncthreads();
  each([&](const Key& k) {
    if (k.a == 0 || better(bound, k)) return;
    const int at = atomicAdd(&L.count, 1);
    if (at < kCap) L.list[at] = k;
  });
  __syncthreads();
  return L.count;
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
  int first;          // row (text) of the launch's first workgroup
};

__device__ __forceinline__ Key1 key_of(float v, int i) {
  return Key1{(static_cast<uint64_t>(score_key_asc(v)) << 32) | (0xffffffffu - static_cast<uint32_t>(i))};
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
  const float mine = top;
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
  float bound = mine;
  {
    int size = 64;
    while (size > 1 && kThreads / size < a.n) size >>= 1;
    for (int o = 1; o < size; o <<= 1) bound = fmaxf(bound, __shfl_xor(bound, o));
    for (int o = size; o < 64; o <<= 1) bound = fminf(bound, __shfl_xor(bound, o));
    __syncthreads();  // red is read
    if (lane == 0) red[wave] = bound;
    if (tid == 0) lists.count = 0;
    __syncthreads();
    bound = fminf(fminf(red[0], red[1]), fminf(red[2], red[3]));
  }
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
  if (c <= kCap) {
    ranked(a.n, c, lists, put);
    return;
  }
  // more equal ones than the list holds (masked rows): by value and index
  Key1 best{0};
  each([&](const Key1& k) {
    if (better(k, best)) best = k;
  });
  c = collected(bound_of(best, a.n, lists.part), lists, each);
  if (c <= kCap) ranked(a.n, c, lists, put);
  else one_by_one(a.n, lists, each, put);
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
__device__ __forceinline__ float key_float(uint32_t k) {
  return __uint_as_float(k >> 31 ? k & 0x7fffffffu : ~k);
}

__global__ __launch_bounds__(kThreads) void beam_join_kernel(BeamArgs a) {
  __shared__ Lists<Key2> lists;
  // x - top first: a row whose tokens are all masked by the type's lowest value is even
  __shared__ double shift[kMaxBeams];  // score - ln sum e^(x - top)
  __shared__ float tops[kMaxBeams];
  const int tid = threadIdx.x, b = a.first + blockIdx.x;
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
  const int per = a.chunks * a.n, all = a.W * per;
  const uint2* pairs = a.pairs + static_cast<int64_t>(b) * all;
  auto key_at = [&](int i) {
    const int w = i / per, j = i - w * per;
    const double s = shift[w];
    if (!(fabs(s) < INFINITY))  // all of the beam's continuations are equal: its first ones
      return j < a.n && j < a.V ? Key2{double_key(s), 0xffffffffu - static_cast<uint32_t>(w * a.V + j)} : Key2{0, 0};
    const uint2 p = pairs[i];
    if (p.x == 0) return Key2{0, 0};
    return Key2{double_key(static_cast<double>(key_float(p.x)) - static_cast<double>(tops[w]) + s),
                0xffffffffu - static_cast<uint32_t>(w * a.V + static_cast<int>(0xffffffffu - p.y))};
  };
  auto each = [&](auto&& f) {
    for (int i = tid; i < all; i += kThreads) f(key_at(i));
  };
  auto put = [&](int rank, const Key2& k) {
    const int flat = static_cast<int>(0xffffffffu - k.b), w = flat / a.V;
    const int64_t at = static_cast<int64_t>(b) * a.n + rank;
    a.out_scores[at] = static_cast<float>(key_double(k.a));
    a.beams[at] = w;
    a.tokens[at] = flat - w * a.V;
    a.parents[at] = b * a.W + w;
  };
  if (all <= kCap) {
    for (int i = tid; i < all; i += kThreads) lists.list[i] = key_at(i);
    __syncthreads();
    ranked(a.n, all, lists, put);
    return;
  }
  Key2 best{0, 0};
  each([&](const Key2& k) {
    if (better(k, best)) best = k;
  });
  const int c = collected(bound_of(best, a.n, lists.part), lists, each);
  if (c <= kCap) ranked(a.n, c, lists, put);
  else one_by_one(a.n, lists, each, put);
}

// Elements of a thread: the longest chunks that leave every CU two workgroups.
int elements_of(int64_t rows, int64_t V) {
  for (int e = 32; e > 8; e /= 2)
    if (rows * ((V + e * kThreads - 1) / (e * kThreads)) >= 2 * device_cus()) return e;
  return 8;
}

// A row that begins inside 16 bytes reaches up to 7 elements further.
int64_t chunks_of(int64_t rows, int64_t V) {
  const int64_t c = static_cast<int64_t>(elements_of(rows, V)) * kThreads;
  return (V + 7 + c - 1) / c;
}

int check_beam(int64_t B, int64_t W, int64_t V, int64_t n, int dtype) {
  HYDRA_REQUIRE(B >= 0 && W >= 1 && V >= 1 && n >= 1, "beam_select: bad size");
  HYDRA_REQUIRE(W <= kMaxBeams && n <= kMaxCount, "beam_select: at most 1024 beams and 128 continuations of a text");
  HYDRA_REQUIRE(V < (int64_t(1) << 31) && W * V < (int64_t(1) << 31) && n <= W * V,
                "beam_select: continuations must be at most beams x vocabulary, and these below 2^31");
  HYDRA_REQUIRE(dtype_size(dtype) > 0, "beam_select: unknown dtype");
  HYDRA_REQUIRE(B < (int64_t(1) << 31) / W && W * chunks_of(B * W, V) * n < (int64_t(1) << 31), "beam_select: too large");
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
    else if (e == 16) beam_chunk_kernel<T, 16><<<grid, kThreads, 0, st>>>(a);
    else beam_chunk_kernel<T, 8><<<grid, kThreads, 0, st>>>(a);
  }
  constexpr int64_t most = int64_t(1) << 22;  // HIP counts a launch's threads in 32 bits
  for (int64_t b = 0; b < a.B; b += most) {
    a.first = static_cast<int>(b);
    beam_join_kernel<<<static_cast<unsigned>(a.B - b < most ? a.B - b : most), kThreads, 0, st>>>(a);
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
  const int64_t rows = B * W, chunks = B == 0 ? 0 : chunks_of(rows, V);
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
  const int64_t rows = B * W, chunks = chunks_of(rows, V);
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
  auto st = static_cast<hipStream_t>(stream);
  return HYDRA_DISPATCH_DTYPE(dtype, T, [&]() -> int { return launch_beam<T>(a, elements_of(rows, V), st); });
}
