// Log probabilities of given tokens, the entropy and the top alternatives of
// their rows of logits, forward and backward, gfx950.
//
// With c = log2(e) / temperature, M = max_j x_j, t_j = (x_j - M) c (the
// difference first: right also where every logit is the type's lowest value),
// s = sum 2^t_j, w = sum 2^t_j t_j,
//   logp_j  = (x_j - M) / T - ln2 log2 s, entropy = ln2 (log2 s - w / s),
//   dL/dx_j = 2^t_j (A + B t_j) + ([j = token] g_lp + sum_k [j = i_k] g_k) / T,
//   B = -ln2 g_H / (s T),  A = -(g_lp + sum_k g_k + g_H (H - ln2 log2 s)) / (s T).
// All of it in fp32; gradients are rounded once.  The backward needs M, s and H
// of a row and no sum over it: it is elementwise.
//
// Both directions are bound by HBM: the forward reads a row once and keeps it
// in registers between its maximum and its sums (16-bit values packed), the
// backward reads it once and writes the gradient.  Rows start anywhere: a row
// is taken in the 16-byte pieces of memory that it lies in, its first and last
// piece element by element where they are not whole.
#include "common.h"
#include "mod_keys.h"

namespace hydra {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// exp2 of anything below is 0; keeps 0 * t_j a 0 where x_j is -inf.
constexpr float kLowest = -2000.f;
constexpr int kThreads = 512;
constexpr int kMaxTop = 64;
constexpr int kCandidates = 1024;

struct LogpArgs {
  const void* x;
  int64_t rs;
  const int64_t* tokens;
  float *logp, *entropy, *stats;  // stats [rows][2]: M, s
  float* top;                     // [rows][K]
  int64_t* top_tokens;
  int V, K;
  float c, inv_t;  // log2(e) / temperature, 1 / temperature
};

// A row as 16-byte pieces of memory: piece i holds the elements E i - shift + (0 .. E-1).
template <typename T>
struct Pieces {
  static constexpr int E = Vec<T>::N;
  const T* x;
  int V, shift, count;
  __device__ __forceinline__ Pieces(const T* row, int v) : x(row), V(v) {
    shift = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
    count = (V + shift + E - 1) / E;
  }
  // Elements outside the row are -inf.
  template <bool NT>
  __device__ __forceinline__ uint4 load(int i) const {
    const int e = i * E - shift;
    if (e >= 0 && e + E <= V) return ld16raw<NT>(x + e);
    float f[E];
#pragma unroll
    for (int k = 0; k < E; ++k) f[k] = e + k >= 0 && e + k < V ? to_f32(x[e + k]) : -INFINITY;
    return pack16<T>(f);  // exact: T's own values
  }
};

template <int N>
__device__ __forceinline__ float max_of(const float* v) {
  float m = v[0];
#pragma unroll
  for (int i = 1; i < N; ++i) m = fmaxf(m, v[i]);
  return m;
}

// Adds a piece's 2^t and 2^t t to s and w.
template <int N>
__device__ __forceinline__ void add_sums(const float* v, float c, float M, float& s, float& w) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    // a NaN stays one: fmaxf would drop it
    const float t = (v[i] - M) * c, u = t < kLowest ? kLowest : t, e = __builtin_amdgcn_exp2f(u);
    s += e;
    w = fmaf(e, u, w);
  }
}

// Order of the alternatives: value down, index up.
__device__ __forceinline__ uint64_t rank_key(float v, int e) {
  return (static_cast<uint64_t>(score_key_asc(v)) << 32) | (0xffffffffu - static_cast<uint32_t>(e));
}

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int off) {
  const uint32_t lo = __shfl_xor(static_cast<uint32_t>(v), off), hi = __shfl_xor(static_cast<uint32_t>(v >> 32), off);
  return (static_cast<uint64_t>(hi) << 32) | lo;
}

// One row per workgroup.  NCH > 0: its pieces stay in registers, NCH of a
// thread; NCH = 0: read again for the sums (rows of more than 16384 pieces).
//
// Alternatives: 64 groups of 8 lanes keep their maximum; the K-th largest of
// these is a bound that at least K elements reach, and few more (about
// 64 ln(64 / (64 - K)) of them where the order is random: 24 for K = 20).
// They are listed in LDS and ranked against each other.  Where equal values
// make them too many, the K best are taken one by one instead.
template <typename T, int NCH, bool TOP>
__global__ __launch_bounds__(kThreads) void logp_kernel(LogpArgs a) {
  constexpr int E = Vec<T>::N, WAVES = kThreads / 64;
  __shared__ float red[2][WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.rs;
  const Pieces<T> pieces(x, a.V);
  uint4 raw[NCH > 0 ? NCH : 1];
  // every piece of this thread's: f(values, first element's index)
  auto each = [&](auto f) {
    if constexpr (NCH > 0) {
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        // the pieces stay packed between the passes: no widened copies kept
        asm volatile("" : "+v"(raw[i].x), "+v"(raw[i].y), "+v"(raw[i].z), "+v"(raw[i].w));
        const int at = i * kThreads + tid;
        if (at < pieces.count) {
          float v[E];
          unpack16<T>(raw[i], v);
          f(v, at * E - pieces.shift);
        }
      }
    } else {
      for (int at = tid; at < pieces.count; at += kThreads) {
        float v[E];
        unpack16<T>(pieces.template load<false>(at), v);
        f(v, at * E - pieces.shift);
      }
    }
  };
  if constexpr (NCH > 0) {
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int at = i * kThreads + tid;
      if (at < pieces.count) raw[i] = pieces.template load<true>(at);
    }
  }
  float m = -INFINITY;
  bool nan = false;
  each([&](const float* v, int) {
    m = fmaxf(m, max_of<E>(v));
    if constexpr (TOP) {
#pragma unroll
      for (int i = 0; i < E; ++i) nan |= v[i] != v[i];
    }
  });
  const float mine = m;
  m = wave_max(m);
  if (lane == 0) red[0][wave] = m;
  __syncthreads();
  m = max_of<WAVES>(red[0]);
  const bool empty = m == -INFINITY;   // nothing is left (or NaN alone, which the sums keep)
  const float M = empty ? 0.f : m;
  float s = 0.f, w = 0.f;
  each([&](const float* v, int) { add_sums<E>(v, a.c, M, s, w); });
  s = wave_sum(s);
  w = wave_sum(w);
  __syncthreads();
  if (lane == 0) {
    red[0][wave] = s;
    red[1][wave] = w;
  }
  __syncthreads();
  s = w = 0.f;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) {
    s += red[0][i];
    w += red[1][i];
  }
  // x = -inf alone: every 2^t is exp2(kLowest) = 0, s = 0
  const float ls = __log2f(s);
  if (tid == 0) {
    const int64_t t = a.tokens[row];
    const bool given = t >= 0 && t < a.V;
    float lp = 0.f;
    if (given) lp = s == 0.f ? -INFINITY : (to_f32(x[t]) - M) * a.inv_t - ls * kLn2;
    a.logp[row] = lp;
    a.entropy[row] = s == 0.f ? 0.f : (ls - w / s) * kLn2;
    if (a.stats) {
      a.stats[2 * row] = M;
      a.stats[2 * row + 1] = s;
    }
  }
  if constexpr (TOP) {
    __shared__ uint32_t bound_s;
    __shared__ int count_s;
    __shared__ uint32_t group[64];
    __shared__ uint64_t list[kCandidates];
    uint32_t key = nan ? 0xffffffffu : score_key_asc(mine);
#pragma unroll
    for (int off = 1; off < kThreads / 64; off <<= 1) key = max(key, static_cast<uint32_t>(__shfl_xor(key, off)));
    if (tid % (kThreads / 64) == 0) group[tid / (kThreads / 64)] = key;
    if (tid == 0) count_s = 0;
    __syncthreads();
    if (wave == 0) {  // the K-th largest of the 64 (equal ones by their place)
      const uint32_t g = group[lane];
      int above = 0;
#pragma unroll 8
      for (int i = 0; i < 64; ++i) above += group[i] > g || (group[i] == g && i < lane);
      if (above == a.K - 1) bound_s = g;
    }
    __syncthreads();
    const uint32_t bound = bound_s;
    each([&](const float* v, int e0) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int e = e0 + i;
        if (score_key_asc(v[i]) >= bound && e >= 0 && e < a.V) {
          const int at = atomicAdd(&count_s, 1);
          if (at < kCandidates) list[at] = rank_key(v[i], e);
        }
      }
    });
    __syncthreads();
    const int count = count_s;
    auto put = [&](int place, uint64_t k) {
      const int e = static_cast<int>(0xffffffffu - static_cast<uint32_t>(k));
      a.top_tokens[row * a.K + place] = e;
      a.top[row * a.K + place] = s == 0.f ? -INFINITY : (to_f32(x[e]) - M) * a.inv_t - ls * kLn2;
    };
    if (count <= kCandidates) {
      for (int i = tid; i < count; i += kThreads) {
        const uint64_t k = list[i];
        int above = 0;
        for (int j = 0; j < count; ++j) above += list[j] > k;
        if (above < a.K) put(above, k);
      }
    } else {
      uint64_t last = ~uint64_t(0);
      for (int place = 0; place < a.K; ++place) {
        uint64_t best = 0;
        for (int e = tid; e < a.V; e += kThreads) {
          const uint64_t k = rank_key(to_f32(x[e]), e);
          if (k < last && k > best) best = k;
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) {
          const uint64_t o = shfl_xor64(best, off);
          best = o > best ? o : best;
        }
        __syncthreads();
        if (lane == 0) list[wave] = best;
        __syncthreads();
        best = list[0];
#pragma unroll
        for (int i = 1; i < WAVES; ++i) best = list[i] > best ? list[i] : best;
        if (tid == 0) put(place, best);
        last = best;
      }
    }
  }
}

struct LogpGradArgs {
  const void* x;
  int64_t rs;
  const int64_t* tokens;
  const float *stats, *entropy;
  const float *g_logp, *g_entropy, *g_top;  // any may be null
  const int64_t* top_tokens;
  void* grad;  // [rows][V]
  int V, K, parts;
  float c, inv_t;
};

constexpr int kGradThreads = 256;
constexpr int kGradPieces = 8;  // of a thread

// Workgroup b takes part b % parts of row b / parts: 2048 pieces.
template <typename T, bool VEC>
__global__ __launch_bounds__(kGradThreads) void logp_grad_kernel(LogpGradArgs a) {
  constexpr int E = Vec<T>::N;
  const int64_t row = blockIdx.x / a.parts;
  const int part = blockIdx.x - static_cast<int>(row) * a.parts, tid = threadIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.rs;
  T* out = static_cast<T*>(a.grad) + row * a.V;
  const Pieces<T> pieces(x, a.V);
  const float M = a.stats[2 * row], s = a.stats[2 * row + 1];
  const int64_t token = a.tokens[row];
  const bool given = token >= 0 && token < a.V;
  const float g_lp = a.g_logp && given ? a.g_logp[row] : 0.f;
  const float g_h = a.g_entropy ? a.g_entropy[row] : 0.f;
  float g_all = g_lp;
  if (a.g_top)
    for (int k = 0; k < a.K; ++k) g_all += a.g_top[row * a.K + k];
  const bool none = s == 0.f;  // a row of -inf alone: no gradient
  const float scale = none ? 0.f : -a.inv_t / s;
  const float A = scale * (g_all + (none ? 0.f : g_h * (a.entropy[row] - kLn2 * __log2f(s)))), B = scale * kLn2 * g_h;
  auto slope = [&](float v) {
    const float t = (v - M) * a.c, u = t < kLowest ? kLowest : t;
    return __builtin_amdgcn_exp2f(u) * fmaf(B, u, A);
  };
  const int begin = part * kGradThreads * kGradPieces;
  uint4 raw[kGradPieces];
#pragma unroll
  for (int i = 0; i < kGradPieces; ++i) {
    const int at = begin + i * kGradThreads + tid;
    if (at < pieces.count) raw[i] = pieces.template load<true>(at);
  }
  const int token_piece = given ? static_cast<int>((token + pieces.shift) / E) : -1;
#pragma unroll
  for (int i = 0; i < kGradPieces; ++i) {
    const int at = begin + i * kGradThreads + tid, e = at * E - pieces.shift;
    if (at >= pieces.count) continue;
    float v[E];
    unpack16<T>(raw[i], v);
#pragma unroll
    for (int k = 0; k < E; ++k) v[k] = slope(v[k]);
    if (at == token_piece && !none) {
#pragma unroll
      for (int k = 0; k < E; ++k) v[k] += e + k == token ? g_lp * a.inv_t : 0.f;
    }
    if (VEC && e >= 0 && e + E <= a.V) {
      store16<T, true>(out + e, v);
    } else {
#pragma unroll
      for (int k = 0; k < E; ++k)
        if (e + k >= 0 && e + k < a.V) out[e + k] = from_f32<T>(v[k]);
    }
  }
  if (a.g_top && !none) {  // the alternatives' own values once more, whole
    __syncthreads();
    for (int k = tid; k < a.K; k += kGradThreads) {
      const int64_t e = a.top_tokens[row * a.K + k];
      const int64_t at = (e + pieces.shift) / E;
      if (e < 0 || e >= a.V || at < begin || at >= begin + kGradThreads * kGradPieces) continue;
      const float own = a.g_top[row * a.K + k] + (e == token ? g_lp : 0.f);
      out[e] = from_f32<T>(slope(to_f32(x[e])) + own * a.inv_t);
    }
  }
}

// Positive, finite, and its inverse too.
bool good_temperature(float t) { return t > 0.f && t < INFINITY && kLog2e / t < INFINITY; }

template <typename T, bool TOP>
int launch_logp(const LogpArgs& a, int64_t rows, hipStream_t st) {
  constexpr int E = Vec<T>::N;
  const int64_t most = (static_cast<int64_t>(a.V) + 2 * E - 2) / E;  // pieces, wherever a row starts
  const dim3 grid(static_cast<unsigned>(rows));
#define HYDRA_LOGP(N) logp_kernel<T, N, TOP><<<grid, kThreads, 0, st>>>(a)
  if (most <= 2 * kThreads) HYDRA_LOGP(2);
  else if (most <= 8 * kThreads) HYDRA_LOGP(8);
  else if (most <= 16 * kThreads) HYDRA_LOGP(16);
  else if (most <= 32 * kThreads) HYDRA_LOGP(32);
  else HYDRA_LOGP(0);
#undef HYDRA_LOGP
  return check_launch("token_logprobs");
}

}  // namespace
}  // namespace hydra

using namespace hydra;

extern "C" int hydra_token_logprobs(const void* logits, int64_t rows, int64_t vocab, int64_t logits_rs,
                                    const int64_t* tokens, float temperature, int64_t top_k, float* logprobs,
                                    float* entropy, float* stats, float* top_logprobs, int64_t* top_tokens, int dtype,
                                    void* stream) {
  HYDRA_REQUIRE(rows >= 0 && vocab >= 1, "token_logprobs: bad size");
  HYDRA_REQUIRE(vocab < (int64_t(1) << 30) && rows < (int64_t(1) << 31), "token_logprobs: too large");
  HYDRA_REQUIRE(logits_rs >= 0, "token_logprobs: negative row stride");
  HYDRA_REQUIRE(top_k >= 0 && top_k <= kMaxTop && top_k <= vocab, "token_logprobs: need 0 <= top_k <= min(64, vocab)");
  HYDRA_REQUIRE(good_temperature(temperature), "token_logprobs: temperature must be positive and finite");
  HYDRA_REQUIRE(dtype_size(dtype) > 0, "token_logprobs: unknown dtype");
  if (rows == 0) return HYDRA_OK;
  HYDRA_REQUIRE(logits && tokens && logprobs && entropy && (top_k == 0 || (top_logprobs && top_tokens)),
                "token_logprobs: null pointer");
  HYDRA_REQUIRE(reinterpret_cast<uintptr_t>(logits) % dtype_size(dtype) == 0, "token_logprobs: misaligned logits");
  const LogpArgs a{logits, logits_rs, tokens, logprobs, entropy, stats, top_logprobs, top_tokens,
                   static_cast<int>(vocab), static_cast<int>(top_k), kLog2e / temperature, 1.f / temperature};
  auto st = static_cast<hipStream_t>(stream);
  return HYDRA_DISPATCH_DTYPE(dtype, T, [&]() -> int {
    return top_k > 0 ? launch_logp<T, true>(a, rows, st) : launch_logp<T, false>(a, rows, st);
  });
}

extern "C" int hydra_token_logprobs_bwd(const void* logits, int64_t rows, int64_t vocab, int64_t logits_rs,
                                        const int64_t* tokens, float temperature, int64_t top_k, const float* stats,
                                        const float* entropy, const int64_t* top_tokens, const float* g_logprobs,
                                        const float* g_entropy, const float* g_top, void* grad, int dtype,
                                        void* stream) {
  HYDRA_REQUIRE(rows >= 0 && vocab >= 1, "token_logprobs_bwd: bad size");
  HYDRA_REQUIRE(vocab < (int64_t(1) << 30) && rows < (int64_t(1) << 31), "token_logprobs_bwd: too large");
  HYDRA_REQUIRE(logits_rs >= 0, "token_logprobs_bwd: negative row stride");
  HYDRA_REQUIRE(top_k >= 0 && top_k <= kMaxTop && top_k <= vocab,
                "token_logprobs_bwd: need 0 <= top_k <= min(64, vocab)");
  HYDRA_REQUIRE(good_temperature(temperature), "token_logprobs_bwd: temperature must be positive and finite");
  const int e = dtype_size(dtype);
  HYDRA_REQUIRE(e > 0, "token_logprobs_bwd: unknown dtype");
  if (rows == 0) return HYDRA_OK;
  HYDRA_REQUIRE(logits && tokens && stats && entropy && grad && (!g_top || top_tokens),
                "token_logprobs_bwd: null pointer");
  HYDRA_REQUIRE(reinterpret_cast<uintptr_t>(logits) % e == 0, "token_logprobs_bwd: misaligned logits");
  const int64_t most = (vocab + 2 * (16 / e) - 2) / (16 / e);
  const int64_t parts = (most + kGradThreads * kGradPieces - 1) / (kGradThreads * kGradPieces);
  HYDRA_REQUIRE(rows * parts < (int64_t(1) << 31), "token_logprobs_bwd: too large");
  const LogpGradArgs a{logits, logits_rs, tokens, stats, entropy, g_logprobs, g_entropy, g_top, top_tokens, grad,
                       static_cast<int>(vocab), static_cast<int>(top_k), static_cast<int>(parts),
                       kLog2e / temperature, 1.f / temperature};
  // A piece of the gradient is whole where the logits' is if rows start alike.
  const bool vec = (reinterpret_cast<uintptr_t>(logits) - reinterpret_cast<uintptr_t>(grad)) % 16 == 0 &&
                   (rows <= 1 || (logits_rs - vocab) * e % 16 == 0);
  auto st = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(rows * parts));
  return HYDRA_DISPATCH_DTYPE(dtype, T, [&]() -> int {
    if (vec) logp_grad_kernel<T, true><<<grid, kGradThreads, 0, st>>>(a);
    else logp_grad_kernel<T, false><<<grid, kGradThreads, 0, st>>>(a);
    return check_launch("token_logprobs_bwd");
  });
}
