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
  Key list[2][kCap];
  Key part[kThreads / 64];
  int count[2];
};

// The least of the maxima of n' >= n groups of threads (all 256 take part): at
// least n elements reach it, if there are as many as groups.
template <typename Key>
__device__ __forceinline__ Key bound_of(Key mine, int n, Key* part) {
  int size = 64;  // of a group
  while (size > 1 && kThreads / size < n) size >>= 1;
  for (int off = 1; off < size; off <<= 1) {
    const Key o = shuffled(mine, off);
    if (better(o, mine)) mine = o;
  }
  for (int off = size; off < 64; off <<= 1) {
    const Key o = shuffled(mine, off);
    if (better(mine, o)) mine = o;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = mine;
  __syncthreads();
  for (int w = 0; w < kThreads / 64; ++w)
    if (better(mine, part[w])) mine = part[w];
  return mine;
}

// The n best of the elements that each thread's `each` goes over, best first, to
// put(rank, key); `best` is the thread's own best.  Ranks without an element get none.
template <typename Key, typename Each, typename Put>
__device__ __forceinline__ void top_n(int n, const Key& best, Lists<Key>& L, Each&& each, Put&& put) {
  const int tid = threadIdx.x;
  const Key none{};
  const Key bound = bound_of(best, n, L.part);
  if (tid == 0) L.count[0] = 0;
  __syncthreads();
  each([&](const Key& k) {
    if (k.a == 0 || better(bound, k)) return;
    const int at = atomicAdd(&L.count[0], 1);
    if (at < kCap) L.list[0][at] = k;
  });
  __syncthreads();
  int c = L.count[0];
  if (c > kCap) {  // one after the other: the best below the last
    Key last = none;
    for (int i = 0; i < n; ++i) {
      Key k = none;
      each([&](const Key& x) {
        if ((i == 0 || better(last, x)) && better(x, k)) k = x;
      });
      for (int off = 1; off < 64; off <<= 1) {
        const Key o = shuffled(k, off);
        if (better(o, k)) k = o;
      }
      __syncthreads();
      if ((tid & 63) == 0) L.part[tid >> 6] = k;
      __syncthreads();
      for (int w = 0; w < kThreads / 64; ++w)
        if (better(L.part[w], k)) k = L.part[w];
      if (tid == 0) put(i, k);
      last = k;
    }
    return;
  }
  Key *from = L.list[0], *to = L.list[1];
  int turn = 0;
  // many: a tighter bound, of the list's own elements
  for (int i = 0; i < 4 && c > kThreads && c > 4 * n; ++i) {
    Key k = none;
    for (int j = tid; j < c; j += kThreads)
      if (better(from[j], k)) k = from[j];
    const Key tight = bound_of(k, n, L.part);
    turn ^= 1;
    if (tid == 0) L.count[turn] = 0;
    __syncthreads();
    for (int j = tid; j < c; j += kThreads)
      if (!better(tight, from[j])) to[atomicAdd(&L.count[turn], 1)] = from[j];
    __syncthreads();
    c = L.count[turn];
    Key* const x = from;
    from = to;
    to = x;
  }
  for (int j = tid; j < c; j += kThreads) {
    const Key k = from[j];
    int rank = 0;
    for (int i = 0; i < c; ++i) rank += better(from[i], k);
    if (rank < n) put(rank, k);
  }
  for (int j = c + tid; j < n; j += kThreads) put(j, none);
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
  top = wave_max(top);
  if (lane == 0) red[wave] = top;
  __syncthreads();
  for (int w = 0; w < 4; ++w) top = fmaxf(top, red[w]);
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
        if (i + e >= 0 && i + e < a.V)
          f(Key1{(static_cast<uint64_t>(score_key_asc(v[j * N + e])) << 32) | (0xffffffffu - static_cast<uint32_t>(i + e))});
    }
  };
  Key1 best{0};
  each([&](const Key1& k) {
    if (better(k, best)) best = k;
  });
  uint2* out = a.pairs + at * a.n;
  top_n(a.n, best, lists, each, [&](int rank, const Key1& k) {
    out[rank] = make_uint2(static_cast<uint32_t>(k.a >> 32), static_cast<uint32_t>(k.a));
  });
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
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int b = a.first + blockIdx.x;
  for (int w = wave; w < a.W; w += kThreads / 64) {
    const float* st = a.stats + 2 * (static_cast<int64_t>(b) * a.W + w) * a.chunks;
    float top = -INFINITY;
    for (int c = lane; c < a.chunks; c += 64) top = fmaxf(top, st[2 * c]);
    top = wave_max(top);
    const double ts = top == -INFINITY ? 0.0 : top;
    double sum = 0.0;
    for (int c = lane; c < a.chunks; c += 64) {
      const float m = st[2 * c], l = st[2 * c + 1];
      sum += m == -INFINITY && l == 0.f ? 0.0 : l * exp(m - ts);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
    if (lane == 0) {  // a row of -inf alone has log probabilities -inf
      shift[w] = sum == 0.0 && top == -INFINITY ? -INFINITY : a.scores[static_cast<int64_t>(b) * a.W + w] - log(sum);
      tops[w] = static_cast<float>(ts);
    }
  }
  __syncthreads();
  const int per = a.chunks * a.n, all = a.W * per;
  const uint2* pairs = a.pairs + static_cast<int64_t>(b) * all;
  auto each = [&](auto&& f) {
    for (int i = tid; i < all; i += kThreads) {
      const int w = i / per, j = i - w * per;
      const double s = shift[w];
      if (!(fabs(s) < INFINITY)) {
        // all of the beam's continuations are equal: its first ones
        if (j < a.n && j < a.V) f(Key2{double_key(s), 0xffffffffu - static_cast<uint32_t>(w * a.V + j)});
        continue;
      }
      const uint2 p = pairs[i];
      if (p.x == 0) continue;
      f(Key2{double_key(static_cast<double>(key_float(p.x)) - static_cast<double>(tops[w]) + s),
            0xffffffffu - static_cast<uint32_t>(w * a.V + static_cast<int>(0xffffffffu - p.y))});
    }
  };
  Key2 best{0, 0};
  each([&](const Key2& k) {
    if (better(k, best)) best = k;
  });
  top_n(a.n, best, lists, each, [&](int rank, const Key2& k) {
    const int flat = static_cast<int>(0xffffffffu - k.b), w = flat / a.V;
    const int64_t at = static_cast<int64_t>(b) * a.n + rank;
    a.out_scores[at] = static_cast<float>(key_double(k.a));
    a.beams[at] = w;
    a.tokens[at] = flat - w * a.V;
    a.parents[at] = b * a.W + w;
  });
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
